// b200spEmbedding, b200spEmbeddingGrad: rows of a table by token, and the gradient of the table.
//
// Both are products with a matrix of one entry a row, S: out = alpha S table + beta out, dTable = alpha S^T grad + beta
// dTable.  Neither reuses anything, so both are bound by the bytes of their rows.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "b200sp_tokens.h"
#include "common/rows.cuh"
#include "tokens/common.cuh"
#include "tokens/sort.cuh"

namespace {

using namespace b200sp_tokens;

// ---------------------------------------------------------------- rows of the table

struct EmbedArgs {
    const void *table, *tokens;
    void *out;
    int vocab, width;
    long long ldTable, ldOut;
    int lanes;             // lanes side by side on a row: a power of two, 32 at most
    unsigned perRow;       // pieces of `lanes` vectors that a row has
    unsigned long long pieces;
    Scalars sc;
};

// What bounds it is how much is on the way: four vectors a thread, held as they were read.  16,384 rows of 4096 bf16: 41 us, with two or
// eight vectors 46 and 47.  (Rows off 16 bytes go element by element: 4095 columns take 185.)
constexpr int kEmbedDepth = 4;

// A vector of kN elements of the table's type, as it lies: in words, of which a 16-bit element alone fills half.
template <typename In, int kN> struct RawRow {
    static constexpr int kWords = kN * (int)sizeof(In) < 4 ? 1 : kN * (int)sizeof(In) / 4;
    uint32_t words[kWords];
    __device__ __forceinline__ void Load(const In *from, int left, bool in)
    {
        if constexpr (kN > 1) {
            if (in && left >= kN) {
#pragma unroll
                for (int i = 0; i < kWords; i += 4) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(from) + i / 4);
                    words[i] = v.x, words[i + 1] = v.y, words[i + 2] = v.z, words[i + 3] = v.w;
                }
                return;
            }
        }
        constexpr int kEach = 4 / (int)sizeof(In);
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            words[i] = 0;
#pragma unroll
            for (int j = 0; j < kEach && kEach * i + j < kN; ++j)
                if (in && kEach * i + j < left) words[i] |= Bits(from[kEach * i + j]) << (16 * j);
        }
    }
    __device__ __forceinline__ float At(int i) const
    {
        if constexpr (sizeof(In) == 4) return __uint_as_float(words[i]);
        else return ToFloat(Element(static_cast<uint16_t>(words[i / 2] >> (16 * (i & 1)))));
    }

private:
    static __device__ __forceinline__ uint32_t Bits(float v) { return __float_as_uint(v); }
    static __device__ __forceinline__ uint32_t Bits(__half v) { return __half_as_ushort(v); }
    static __device__ __forceinline__ uint32_t Bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
    static __device__ __forceinline__ In Element(uint16_t v)
    {
        if constexpr (std::is_same_v<In, __half>) return __ushort_as_half(v);
        else return __ushort_as_bfloat16(v);
    }
};

template <typename In, typename Out, typename Key, int kN>
__global__ void __launch_bounds__(256) EmbeddingKernel(const EmbedArgs a)
{
    b200sp::WaitForPrevious();
    constexpr bool kVector = kN > 1;
    const int lane = threadIdx.x & 31;
    const int rowsPerWarp = 32 / a.lanes, sub = lane / a.lanes, at = lane % a.lanes;
    const unsigned long long first = ((unsigned long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kEmbedDepth * rowsPerWarp + sub;
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    RawRow<In, kN> raw[kEmbedDepth];
    long long to[kEmbedDepth];  // -1: nothing
    int left[kEmbedDepth];      // elements of the row from here
    // Rows of several pieces have all lanes on each: one division, then a piece further every time.
    long long row;
    unsigned within;
    if (a.perRow == 1) {
        row = (long long)first;
        within = 0;
    } else if (a.pieces <= UINT_MAX) {
        row = (unsigned)first / a.perRow;
        within = (unsigned)first % a.perRow;
    } else {
        row = (long long)(first / a.perRow);
        within = (unsigned)(first % a.perRow);
    }
#pragma unroll
    for (int u = 0; u < kEmbedDepth; ++u) {
        if (u > 0 && a.perRow == 1) {
            row += rowsPerWarp;
        } else if (u > 0 && ++within == a.perRow) {
            within = 0;
            ++row;
        }
        to[u] = -1;
        if (first + (unsigned long long)u * rowsPerWarp >= a.pieces) continue;
        const int col = (int)(within * a.lanes + at) * kN;
        left[u] = a.width - col;
        if (left[u] <= 0) continue;
        to[u] = row * a.ldOut + col;
        const Key token = __ldg(static_cast<const Key *>(a.tokens) + row);
        const bool in = token >= 0 && token < (Key)a.vocab;
        const In *const from = static_cast<const In *>(a.table) + (long long)(in ? token : 0) * a.ldTable + col;
        raw[u].Load(from, left[u], in);
    }
#pragma unroll
    for (int u = 0; u < kEmbedDepth; ++u) {
        if (to[u] < 0) continue;
        Out *const out = static_cast<Out *>(a.out) + to[u];
        float v[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            v[i] = alpha * raw[u].At(i);
            if (beta != 0.0f && i < left[u]) v[i] = fmaf(beta, ToFloat(out[i]), v[i]);
        }
        if (left[u] >= kN) {
            StoreFloats<Out, kN, kVector>(out, v);
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (i < left[u]) out[i] = FromFloat<Out>(v[i]);
        }
    }
}

// ---------------------------------------------------------------- the gradient of the table

// The positions are sorted by token (sort.cuh), in the same launch as some zeros of dTable: the sort is one cluster's work
// and the zeros everyone else's; the other zeros are written beside the joins, which are few and wait long.  Then a group of lanes takes `chunk` sorted positions and sums their rows of grad, in
// that order, one token after the other.  A token whose positions lie in one chunk is finished there; of one that
// crosses chunks every chunk leaves a partial row, which EmbeddingJoinKernel adds up in their order.
// 16,384 rows of 2048 bf16, a table of 65,536 rows in f32 (604 MB): 119 us; 164 with a part of the zeros beside the sums, whose reads wait
// longer then; 199 with all zeros beside the sort, and rows held as floats, eight deep.  (Zeros alone run at 3.8 TB/s in long stretches, 6.3
// a row per warp.)
struct GradArgs {
    const void *grad;
    void *table;
    int count, vocab, width;
    long long ldGrad, ldTable;
    const int *keys, *positions;  // sorted
    int chunk, chunks;
    float *heads, *tails;         // [chunk][pitch]: of the run that comes from the chunk before, that goes on in the next
    int pitch;
    int lanes;                    // threads side by side on a row
    int fillFirst;                // with beta = 0: rows that get zeros while the tokens are sorted
    unsigned sumBlocks, sumAcross;  // CTAs that sum, and of those side by side on a row
    unsigned fillBlocks;            // of EmbeddingJoinKernel, CTAs beside them that write zeros
    Scalars sc;
};

// Zeros for the first `fillFirst` rows.
template <typename Out> __device__ __forceinline__ void FillTable(const GradArgs &a, int block, int blocks)
{
    Out *const table = static_cast<Out *>(a.table);
    if (a.ldTable == a.width && (reinterpret_cast<uintptr_t>(table) & 15) == 0) {
        const long long elements = (long long)a.fillFirst * a.width, pieces = elements * (long long)sizeof(Out) / 16;
        uint4 *const to = reinterpret_cast<uint4 *>(table);
        const long long step = (long long)blocks * blockDim.x;
        long long i = (long long)block * blockDim.x + threadIdx.x;
        for (; i + 3 * step < pieces; i += 4 * step) {
#pragma unroll
            for (int u = 0; u < 4; ++u) __stcs(to + i + u * step, make_uint4(0, 0, 0, 0));
        }
        for (; i < pieces; i += step) __stcs(to + i, make_uint4(0, 0, 0, 0));
        const long long rest = pieces * (16 / (long long)sizeof(Out)) + threadIdx.x;
        if (block == 0 && rest < elements) table[rest] = FromFloat<Out>(0.0f);
        return;
    }
    for (long long r = block; r < a.fillFirst; r += blocks)  // a step past the last of 2^31 - 2 rows is no int
        for (int c = threadIdx.x; c < a.width; c += blockDim.x) table[r * a.ldTable + c] = FromFloat<Out>(0.0f);
}

// Zeros for the rows after them whose tokens do not occur: a warp per row, some rows each.
constexpr int kFillRows = 4;
template <typename Out> __device__ __forceinline__ void FillOthers(const GradArgs &a, int block)
{
    const int lane = threadIdx.x & 31;
    for (int i = 0; i < kFillRows; ++i) {
        const long long r = (long long)a.fillFirst + ((long long)block * 8 + (threadIdx.x >> 5)) * kFillRows + i;
        if (r >= a.vocab) return;
        const int at = b200sp::WarpLowerBound(a.keys, a.count, r, lane);
        if (at < a.count && __ldg(a.keys + at) == r) continue;
        Out *const row = static_cast<Out *>(a.table) + r * a.ldTable;
        int c = 0;
        if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {
            const int pieces = a.width * (int)sizeof(Out) / 16;
            for (int k = lane; k < pieces; k += 32) __stcs(reinterpret_cast<uint4 *>(row) + k, make_uint4(0, 0, 0, 0));
            c = pieces * (16 / (int)sizeof(Out));
        }
        for (c += lane; c < a.width; c += 32) row[c] = FromFloat<Out>(0.0f);
    }
}

// CTAs that sum wait for what they read, CTAs that fill for nothing: they are mixed evenly.  Whether this one fills, and else which of the
// others it is.
template <typename Out> __device__ __forceinline__ bool FillsInstead(const GradArgs &a, unsigned *block)
{
    const unsigned long long all = (unsigned long long)a.sumBlocks + a.fillBlocks;
    const unsigned fills = (unsigned)(blockIdx.x * (unsigned long long)a.fillBlocks / all);  // before this one
    *block = blockIdx.x - fills;
    if ((blockIdx.x + 1ull) * a.fillBlocks / all == fills) return false;
    if (a.sc.Beta() == 0.0f) FillOthers<Out>(a, (int)fills);
    return true;
}

template <typename Out, typename Key>
__global__ void __launch_bounds__(kSortThreads, 1) EmbeddingSortKernel(const SortArgs s, const GradArgs a, int clusters)
{
    extern __shared__ unsigned char sSort[];
    b200sp::WaitForPrevious();
    const int size = gridDim.x / clusters;
    if ((int)blockIdx.x < size) {
        ClusterSort<Key>(s, sSort, [](int, int, int) {});
    } else if (a.sc.Beta() == 0.0f) {
        FillTable<Out>(a, blockIdx.x - size, gridDim.x - size);
    }
}

// First place of the ascending keys that is >= key.
__device__ __forceinline__ int LowerBound(const int *keys, int count, int key)
{
    int lo = 0, hi = count;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (__ldg(keys + mid) < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// beta other than 0 and 1: rows of tokens that do not occur.  (The rows of those that do are scaled where they are rounded.)
template <typename Out> __global__ void __launch_bounds__(256) EmbeddingScaleKernel(const GradArgs a)
{
    b200sp::WaitForPrevious();
    const float beta = a.sc.Beta();
    if (beta == 0.0f || beta == 1.0f) return;
    for (long long r = blockIdx.x; r < a.vocab; r += gridDim.x) {
        const int at = LowerBound(a.keys, a.count, (int)r);
        if (at < a.count && __ldg(a.keys + at) == r) continue;
        Out *const row = static_cast<Out *>(a.table) + r * a.ldTable;
        for (int c = threadIdx.x; c < a.width; c += 256) row[c] = FromFloat<Out>(beta * ToFloat(row[c]));
    }
}

template <typename Out, int kN> __device__ __forceinline__ void FinishRow(const GradArgs &a, int key, int col, float (&sum)[kN])
{
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    Out *const to = static_cast<Out *>(a.table) + key * a.ldTable + col;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        sum[i] *= alpha;
        if (beta != 0.0f && col + i < a.width) sum[i] = fmaf(beta, ToFloat(to[i]), sum[i]);
    }
    if (col + kN <= a.width) {
        StoreFloats<Out, kN, (kN > 1)>(to, sum);
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (col + i < a.width) to[i] = FromFloat<Out>(sum[i]);
    }
}

constexpr int kGradDepth = 4, kJoinDepth = 8;  // rows, and partial ones, in flight of a thread

template <typename In, typename Out, int kN> __global__ void __launch_bounds__(256) EmbeddingSumKernel(const GradArgs a)
{
    b200sp::WaitForPrevious();
    const int chunk = (int)(blockIdx.x / a.sumAcross) * (256 / a.lanes) + threadIdx.x / a.lanes;
    const int col = (int)(blockIdx.x % a.sumAcross * a.lanes + threadIdx.x % a.lanes) * kN;
    if (chunk >= a.chunks || col >= a.width) return;
    const int lo = chunk * a.chunk, hi = (int)min((long long)a.count, (long long)lo + a.chunk);
    const int before = lo > 0 ? __ldg(a.keys + lo - 1) : -1, after = hi < a.count ? __ldg(a.keys + hi) : -1;
    float sum[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) sum[i] = 0.0f;
    int now = __ldg(a.keys + lo);
    bool continued = now == before;
    auto flush = [&](bool end) {
        if (now < a.vocab) {
            if (continued || (end && now == after)) {
                float *const to = (continued ? a.heads : a.tails) + (long long)chunk * a.pitch + col;
#pragma unroll
                for (int i = 0; i < kN; ++i) to[i] = sum[i];  // the pitch has room for whole vectors
            } else {
                FinishRow<Out, kN>(a, now, col, sum);
            }
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) sum[i] = 0.0f;
        continued = false;
    };
    int key[kGradDepth], position[kGradDepth];  // of the rows to come: -1 none
    auto look = [&](int e) {
#pragma unroll
        for (int u = 0; u < kGradDepth; ++u) {
            key[u] = e + u < hi ? __ldg(a.keys + e + u) : -1;
            position[u] = e + u < hi ? __ldg(a.positions + e + u) : 0;
        }
    };
    look(lo);
    for (int e = lo; e < hi; e += kGradDepth) {
        RawRow<In, kN> v[kGradDepth];
        int token[kGradDepth];
#pragma unroll
        for (int u = 0; u < kGradDepth; ++u) {
            token[u] = key[u];
            if (key[u] >= 0) v[u].Load(static_cast<const In *>(a.grad) + (long long)position[u] * a.ldGrad + col, a.width - col, true);
        }
        look(e + kGradDepth);
#pragma unroll
        for (int u = 0; u < kGradDepth; ++u) {
            if (token[u] < 0) continue;
            if (token[u] != now) {
                flush(false);
                now = token[u];
            }
#pragma unroll
            for (int i = 0; i < kN; ++i) sum[i] += v[u].At(i);
        }
    }
    flush(true);
}

// Tokens whose positions cross chunks: the chunk where one begins adds up what the others left, eight at a time.
template <typename Out, int kN> __global__ void __launch_bounds__(256) EmbeddingJoinKernel(const GradArgs a)
{
    b200sp::WaitForPrevious();
    unsigned block;
    if (FillsInstead<Out>(a, &block)) return;
    const int chunk = (int)(block / a.sumAcross) * (256 / a.lanes) + threadIdx.x / a.lanes;
    const int col = (int)(block % a.sumAcross * a.lanes + threadIdx.x % a.lanes) * kN;
    if (chunk >= a.chunks - 1 || col >= a.width) return;
    const int hi = (chunk + 1) * a.chunk, lo = hi - a.chunk;
    const int key = __ldg(a.keys + hi - 1), next = __ldg(a.keys + hi), before = lo > 0 ? __ldg(a.keys + lo - 1) : -1;
    if (key >= a.vocab || next != key || before == key) return;  // none crosses, or it began before
    float sum[kN];
    const float *at = a.tails + (long long)chunk * a.pitch + col;
#pragma unroll
    for (int i = 0; i < kN; ++i) sum[i] = at[i];
    bool more = true;
    for (int c = chunk + 1; more && c < a.chunks; c += kJoinDepth) {
        float v[kJoinDepth][kN];
        int starts[kJoinDepth];
#pragma unroll
        for (int u = 0; u < kJoinDepth; ++u) {
            const int from = min(c + u, a.chunks - 1);
            starts[u] = c + u < a.chunks ? __ldg(a.keys + from * a.chunk) : -1;
            const float *heads = a.heads + (long long)from * a.pitch + col;
#pragma unroll
            for (int i = 0; i < kN; ++i) v[u][i] = heads[i];
        }
#pragma unroll
        for (int u = 0; u < kJoinDepth; ++u) {
            more = more && starts[u] == key;  // the chunk begins with this token: its head is a piece of it
#pragma unroll
            for (int i = 0; i < kN; ++i) sum[i] = more ? sum[i] + v[u][i] : sum[i];
        }
    }
    FinishRow<Out, kN>(a, key, col, sum);
}

// ---------------------------------------------------------------- host

aclsparseStatus_t CheckTokens(const aclsparseDnVecDescr *tokens)
{
    if (tokens == nullptr || tokens->magic != b200sp::kDnVecMagic) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (tokens->valueType != ACL_INT32 && tokens->valueType != ACL_INT64) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (tokens->size > kMostCounted) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (!OnBoundary(tokens->values, tokens->valueType == ACL_INT64 ? 8 : 4)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

// The rows that a call reads or writes, and the tokens that name them.
aclsparseStatus_t CheckEmbedding(const aclsparseDnMatDescr *table, const aclsparseDnVecDescr *tokens, const aclsparseDnMatDescr *rows)
{
    for (const aclsparseDnMatDescr *m : {table, rows}) {
        const aclsparseStatus_t st = CheckDense(m);
        if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    }
    const aclsparseStatus_t st = CheckTokens(tokens);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (rows->rows != tokens->size || rows->cols != table->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (table->rows >= INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;  // the number after the last row is a key, too
    return ACL_SPARSE_STATUS_SUCCESS;
}

int LanesFor(long long vectors, int most)
{
    int lanes = 1;
    while (lanes < most && lanes < vectors) lanes *= 2;
    return lanes;
}

// Chunks of the gradient.  Long ones leave fewer partial rows, short ones fill the SMs.  bf16 gradients of 32,000 x 1024 f32, us with chunks of
// 8 and 32 positions: 512 tokens 29 and 38, 2048 30 and 37, 4096 33 and 37, 8192 46 and 48, 12,288 57 and 50, 16,384 64 and 53.
int ChunkFor(long long count)
{
    int chunk = count <= 8192 ? 8 : 32;
    while (count > 4096ll * chunk) chunk *= 2;
    return chunk;
}

struct GradLayout {
    size_t keyA, posA, keyB, posB, heads, tails, total;
    int chunk, chunks, pitch;
};
GradLayout GradLayoutFor(long long count, long long width)
{
    GradLayout L;
    const size_t words = AlignUp(sizeof(int) * (size_t)count, 256);
    L.keyA = 0;
    L.posA = words;
    L.keyB = 2 * words;
    L.posB = 3 * words;
    L.heads = 4 * words;
    L.chunk = ChunkFor(count);
    L.chunks = (int)((count + L.chunk - 1) / L.chunk);
    L.pitch = (int)AlignUp((size_t)width, 64);
    const size_t partial = sizeof(float) * (size_t)L.chunks * (size_t)L.pitch;
    L.tails = L.heads + partial;
    L.total = L.tails + partial + 256;  // any address is accepted
    return L;
}

template <typename In, typename Out, typename Key, int kN> cudaError_t LaunchEmbedding(EmbedArgs a, long long rows, cudaStream_t stream)
{
    const long long vectors = (a.width + kN - 1) / kN;
    a.lanes = LanesFor(vectors, 32);
    a.perRow = (unsigned)((vectors + a.lanes - 1) / a.lanes);
    a.pieces = (unsigned long long)rows * a.perRow;
    const unsigned long long perBlock = 8ull * kEmbedDepth * (32 / a.lanes), blocks = (a.pieces + perBlock - 1) / perBlock;
    if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    b200sp_note_launches(1);
    return b200sp::LaunchChained(EmbeddingKernel<In, Out, Key, kN>, (unsigned)blocks, 256, 0, stream, a);
}

template <typename In, typename Out, int kN> cudaError_t LaunchSums(GradArgs a, bool scales, cudaStream_t stream)
{
    if (scales) {
        b200sp_note_launches(1);
        const cudaError_t e = b200sp::LaunchChained(EmbeddingScaleKernel<Out>, (unsigned)std::min(a.vocab, b200sp_sm_count() * 8), 256, 0, stream, a);
        if (e != cudaSuccess) return e;
    }
    const long long vectors = (a.width + kN - 1) / kN;
    a.lanes = LanesFor(vectors, 256);
    const int perBlock = 256 / a.lanes;
    const long long across = (vectors + a.lanes - 1) / a.lanes, sums = (a.chunks + perBlock - 1) / perBlock * across;
    const bool fills = a.sc.betaAt != nullptr || a.sc.beta == 0.0f;
    const long long others = fills ? ((long long)a.vocab - a.fillFirst + 8 * kFillRows - 1) / (8 * kFillRows) : 0;
    if (sums + others > INT32_MAX) return cudaErrorInvalidConfiguration;
    a.sumAcross = (unsigned)across;
    a.sumBlocks = (unsigned)sums;
    a.fillBlocks = (unsigned)others;
    b200sp_note_launches(2);
    const cudaError_t e = b200sp::LaunchChained(EmbeddingSumKernel<In, Out, kN>, (unsigned)sums, 256, 0, stream, a);
    return e != cudaSuccess ? e : b200sp::LaunchChained(EmbeddingJoinKernel<Out, kN>, (unsigned)(sums + others), 256, 0, stream, a);
}

// Rows that are filled while the tokens are sorted: what is written in that time.  16,384 tokens of 65,536 x 2048 f32: 64 MB 119 us, none 125, 128
// MB 127; 2048 tokens of 32,000 x 1024: 31, 36, 32.  Rows of less than 1024 bytes all are: to look up whether a token occurs costs more than to
// write them where there are many (20,000 tokens of 1,500,000 x 16 f32: 48 us, looked up 136; 4096 tokens of 500,000 x 64: 31 and 71; with
// 131,072 rows of 512 bytes 23 and 23, of 2048 bytes 55 and 49).
constexpr long long kFillAhead = 64 << 20;
int FillFirst(long long vocab, long long rowBytes)
{
    return (int)(rowBytes < 1024 ? vocab : std::min(vocab, std::max(1ll, kFillAhead / rowBytes)));
}

template <typename Out, typename Key> cudaError_t LaunchSort(const SortArgs &s, const GradArgs &a, cudaStream_t stream)
{
    const int size = SortCtas(a.count), shared = SortShared(s.digitBits, a.count <= kSortTile && s.passes > 1);
    const cudaError_t set = AllowShared<EmbeddingSortKernel<Out, Key>>(kSortSharedMost);
    if (set != cudaSuccess) return set;
    // one cluster sorts; the others fill the table, if it has to be (one CTA per SM: what the sort needs of shared memory)
    const bool fills = a.sc.betaAt != nullptr || a.sc.beta == 0.0f;
    const int clusters = fills ? std::max(2, b200sp_sm_count() / size) : 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(size * clusters));
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = (size_t)shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)size;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    b200sp_note_launches(1);
    return cudaLaunchKernelEx(&cfg, EmbeddingSortKernel<Out, Key>, s, a, clusters);
}

}  // namespace

extern "C" {

aclsparseStatus_t b200spEmbedding(aclsparseHandle_t handle, const void *alpha, aclsparseConstDnMatDescr_t table,
                                  aclsparseConstDnVecDescr_t tokens, const void *beta, aclsparseDnMatDescr_t out)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    const aclsparseStatus_t st = CheckEmbedding(table, tokens, out);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const OnDevice device(handle);
    EmbedArgs a{table->values, tokens->values, out->values, (int)table->rows, (int)table->cols, table->ld, out->ld, 0, 0, 0,
                ScalarsOf(handle, alpha, beta)};
    const bool vectors = RowsAligned(table) && RowsAligned(out);
    const cudaError_t e = WithType(table->valueType, [&](auto in) {
        return WithType(out->valueType, [&](auto to) {
            using In = decltype(in);
            using Out = decltype(to);
            // 16 bytes of the narrower type
            constexpr int kN = sizeof(In) == 2 || sizeof(Out) == 2 ? 8 : 4;
            if (tokens->valueType == ACL_INT64)
                return vectors ? LaunchEmbedding<In, Out, long long, kN>(a, out->rows, handle->stream)
                               : LaunchEmbedding<In, Out, long long, 1>(a, out->rows, handle->stream);
            return vectors ? LaunchEmbedding<In, Out, int, kN>(a, out->rows, handle->stream)
                           : LaunchEmbedding<In, Out, int, 1>(a, out->rows, handle->stream);
        });
    });
    return Finished(e, "b200spEmbedding");
}

aclsparseStatus_t b200spEmbeddingGradBufferSize(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t grad,
                                                aclsparseConstDnVecDescr_t tokens, aclsparseConstDnMatDescr_t dTable,
                                                size_t *bufferSize)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckEmbedding(dTable, tokens, grad);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    *bufferSize = GradLayoutFor(tokens->size, dTable->cols).total;
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t b200spEmbeddingGrad(aclsparseHandle_t handle, const void *alpha, aclsparseConstDnMatDescr_t grad,
                                      aclsparseConstDnVecDescr_t tokens, const void *beta, aclsparseDnMatDescr_t dTable,
                                      void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    const aclsparseStatus_t st = CheckEmbedding(dTable, tokens, grad);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    const OnDevice device(handle);
    (void)NoteWrite(buffer);
    const GradLayout L = GradLayoutFor(tokens->size, dTable->cols);
    char *const p = reinterpret_cast<char *>(AlignUp(reinterpret_cast<uintptr_t>(buffer), 256));
    SortArgs s{};
    s.keys = tokens->values;
    s.count = (int)tokens->size;
    s.limit = (int)dTable->rows;
    SortPasses(s.limit, s.count, &s);
    s.keyA = reinterpret_cast<int *>(p + L.keyA);
    s.posA = reinterpret_cast<int *>(p + L.posA);
    s.keyB = reinterpret_cast<int *>(p + L.keyB);
    s.posB = reinterpret_cast<int *>(p + L.posB);
    GradArgs a{};
    a.grad = grad->values;
    a.table = dTable->values;
    a.count = s.count;
    a.vocab = s.limit;
    a.width = (int)dTable->cols;
    a.ldGrad = grad->ld;
    a.ldTable = dTable->ld;
    a.keys = s.keyA;
    a.positions = s.posA;
    a.chunk = L.chunk;
    a.chunks = L.chunks;
    a.heads = reinterpret_cast<float *>(p + L.heads);
    a.tails = reinterpret_cast<float *>(p + L.tails);
    a.pitch = L.pitch;
    a.fillFirst = FillFirst(dTable->rows, dTable->cols * BytesOf(dTable->valueType));
    a.sc = ScalarsOf(handle, alpha, beta);
    const bool scales = a.sc.betaAt != nullptr || (a.sc.beta != 0.0f && a.sc.beta != 1.0f);
    const bool vectors = RowsAligned(grad) && RowsAligned(dTable);
    const cudaError_t e = WithType(dTable->valueType, [&](auto to) {
        using Out = decltype(to);
        const cudaError_t sorted = tokens->valueType == ACL_INT64 ? LaunchSort<Out, long long>(s, a, handle->stream)
                                                                  : LaunchSort<Out, int>(s, a, handle->stream);
        if (sorted != cudaSuccess) return sorted;
        return WithType(grad->valueType, [&](auto from) {
            using In = decltype(from);
            constexpr int kN = sizeof(In) == 2 || sizeof(Out) == 2 ? 8 : 4;
            return vectors ? LaunchSums<In, Out, kN>(a, scales, handle->stream) : LaunchSums<In, Out, 1>(a, scales, handle->stream);
        });
    });
    return Finished(e, "b200spEmbeddingGrad");
}

}  // extern "C"
