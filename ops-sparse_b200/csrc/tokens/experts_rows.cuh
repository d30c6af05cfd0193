// Rows of tokens in the order of their experts, and back: included by experts.cu.
//
// dispatch: S[place(i)] = alpha X[token(i)]; combine: out[t] = alpha sum of w_i S[place(i)]; its gradient: dS[place(i)] = alpha w_i dOut[t],
// dw_i = alpha <dOut[t], S[place(i)]>.  All go by tokens, whose entries lie side by side in R: a token's row is read (or written) once and stays in
// registers while the rows of its entries, which lie anywhere, are written (or read).  What bounds dispatch and combine is DRAM; neighbouring warps take neighbouring
// stretches of a row, so that a row is read or written as a whole at about one time.
// One B200, bf16, us (the bytes at the copy rate of 6550 GB/s in brackets): rows of 8192 tokens of 4096 to four of 32 experts 57 (51); the weighted sum of eight
// of 64 experts' rows of 2048 for 8192 tokens 57 (46); its gradient, four of 32, 64 (46); one token's eight rows 4, which is a launch and the host's call.
#pragma once

struct RowsArgs {
    const int4 *header;  // as in MmaArgs
    int4 mark;
    uint64_t number;
    const int *offsets, *places;
    const int *rowPtr;
    long long tokens;
    int nnz, experts, width;
    const void *perToken, *perEntry;  // read
    void *out;                        // written: a row per token or per entry
    long long ldToken, ldEntry, ldOut;
    const void *weights;              // nullptr: none
    aclDataType weightType;
    void *dValues;                    // nullptr: none
    aclDataType dValuesType;
    float *scales;
    int *starts;                      // nullptr, or [experts + 1]: the first row of every expert
    Scalars sc;
};

// Rounding to 8 bits lets the next kernel in early (a product takes every SM, and keeps other streams from them while it waits) only where it is a matter of some us:
// by half of the SMs, rows that are held, and so many stretches of rows to be written, eight of a row at least, all by one CTA at worst, 18 us (f32 23).  16 tokens
// to eight of 64 experts, order, rounding and product 32.1 us, without 32.6; one row of 4096 and its product 6.57 and 6.7.  (The order of the entries, by eight SMs,
// does not: one of 1,048,576 entries takes 285 us, in which another stream's product ends in 17, and not in 440; behind orders of 8 to 32,768 entries nothing is
// gained.)
constexpr unsigned kFewCtas = 74;
constexpr long long kFewPieces = 2048;
constexpr int kRowsThreads = 256, kRowsWarps = kRowsThreads / 32;
constexpr int kDispatchCtas = 5, kCombineCtas = 4, kGradCtas = 2;  // resident on an SM: what their registers allow
template <typename T> constexpr int kQuantiseCtas = sizeof(T) == 4 ? 4 : 6;

// What every call of this file ends its beginning with: false without an order.  What has been read of the buffer by then (places may be any
// numbers) leads to no access.
__device__ __forceinline__ bool HasOrder(const RowsArgs &a)
{
    if (!StartsWith(a.header, a.mark, a.number)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicMax(&gExpertsError, kNoOrder);
        return false;
    }
    if (a.starts != nullptr && blockIdx.x == gridDim.x - 1)
        for (int e = threadIdx.x; e <= a.experts; e += kRowsThreads) a.starts[e] = __ldg(a.offsets + e);
    return true;
}
// The entries of a token, whatever the offsets say.
__device__ __forceinline__ int2 EntriesOf(const RowsArgs &a, long long token)
{
    return make_int2(max(0, __ldg(a.rowPtr + token)), min(a.nnz, __ldg(a.rowPtr + token + 1)));
}

// (A row's pitch has 31 bits, so that this is one multiplication.)
template <typename T> __device__ __forceinline__ T *RowAt(T *rows, int row, long long pitch) { return rows + (long long)row * (int)pitch; }

// The entries of a token, and where the rows of the first 32 lie, a lane each; asked for ahead of the rows.
struct TokenEntries {
    int2 range;
    int place;
    float weight;
    __device__ __forceinline__ void Rows(const RowsArgs &a, int e0, int lane)
    {
        place = 0;
        weight = 1.0f;
        if (e0 + lane < range.y) {
            place = __ldg(a.places + e0 + lane);
            if (a.weights != nullptr) weight = ValueAt(a.weights, a.weightType, e0 + lane);
        }
    }
    __device__ __forceinline__ void Ask(const RowsArgs &a, long long token, int lane)
    {
        range = token < a.tokens ? EntriesOf(a, token) : make_int2(0, 0);
        Rows(a, range.x, lane);
    }
};

template <typename In, typename Out, bool kVector>
__global__ void __launch_bounds__(kRowsThreads, kDispatchCtas) ExpertsDispatchKernel(const RowsArgs a)
{
    b200sp::WaitForPrevious();
    const int lane = threadIdx.x & 31, end = __ldg(a.offsets + a.experts);
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    Units u((long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5), (long long)gridDim.x * kRowsWarps, (a.width + kStretch - 1) / kStretch);
    TokenEntries next;
    next.Ask(a, u.row, lane);
    if (!HasOrder(a)) return;
    while (u.row < a.tokens) {
        const int c0 = u.stretch * kStretch;
        Raw<In> raw;
        raw.template Load<kVector>(static_cast<const In *>(a.perToken) + u.row * a.ldToken, c0, lane, a.width);
        TokenEntries now = next;
        u.Next();
        next.Ask(a, u.row, lane);
        float v[8];
        raw.Floats(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= alpha;
        Raw<Out> row, none;
        row.Set(v);
        none.Zero();
        for (int e0 = now.range.x; e0 < now.range.y; e0 += 32) {
            if (e0 > now.range.x) now.Rows(a, e0, lane);
            const int many = min(32, now.range.y - e0);
            for (int j = 0; j < many; ++j) {
                const int place = __shfl_sync(0xffffffffu, now.place, j);
                Out *const to = RowAt(static_cast<Out *>(a.out), place, a.ldOut);
                if (beta == 0.0f) {
                    if (place < end) row.template Store<kVector>(to, c0, lane, a.width);
                    else none.template Store<kVector>(to, c0, lane, a.width);
                } else {
                    Raw<Out> old;
                    old.template Load<kVector>(to, c0, lane, a.width);
                    float w[8];
                    old.Floats(w);
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = fmaf(beta, w[i], place < end ? v[i] : 0.0f);
                    old.Set(w);
                    old.template Store<kVector>(to, c0, lane, a.width);
                }
            }
        }
    }
}

// Rows are asked for kAhead at a time, and the places of the next unit's before this one's are summed: one row after the other, by a grid of more CTAs than the
// SMs hold, took 87 us where this takes 57.  (The next unit's rows brought to L2 ahead: 61.)
template <typename In, typename Out, bool kVector>
__global__ void __launch_bounds__(kRowsThreads, kCombineCtas) ExpertsCombineKernel(const RowsArgs a)
{
    constexpr int kAhead = sizeof(In) == 4 ? 2 : 4;
    b200sp::WaitForPrevious();
    const int lane = threadIdx.x & 31, end = __ldg(a.offsets + a.experts);
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    Units u((long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5), (long long)gridDim.x * kRowsWarps, (a.width + kStretch - 1) / kStretch);
    TokenEntries next;
    next.Ask(a, u.row, lane);
    if (!HasOrder(a)) return;
    while (u.row < a.tokens) {
        const int c0 = u.stretch * kStretch;
        const long long token = u.row;
        TokenEntries now = next;
        u.Next();
        next.Ask(a, u.row, lane);
        float sum[8] = {};
        for (int e0 = now.range.x; e0 < now.range.y; e0 += 32) {
            if (e0 > now.range.x) now.Rows(a, e0, lane);
            const int many = min(32, now.range.y - e0);
            for (int j0 = 0; j0 < many; j0 += kAhead) {
                Raw<In> raw[kAhead];
                bool in[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const int place = __shfl_sync(0xffffffffu, now.place, (j0 + j) & 31);
                    in[j] = j0 + j < many && place < end;
                    if (in[j]) raw[j].template Load<kVector>(RowAt(static_cast<const In *>(a.perEntry), place, a.ldEntry), c0, lane, a.width);
                }
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const float w = __shfl_sync(0xffffffffu, now.weight, (j0 + j) & 31);
                    if (in[j]) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) sum[i] = fmaf(w, raw[j].At(i), sum[i]);
                    }
                }
            }
        }
        Out *const to = static_cast<Out *>(a.out) + token * a.ldOut;
        Raw<Out> out;
        if (beta != 0.0f) {
            out.template Load<kVector>(to, c0, lane, a.width);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = fmaf(beta, out.At(i), alpha * sum[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] *= alpha;
        }
        out.Set(sum);
        out.template Store<kVector>(to, c0, lane, a.width);
    }
}

// T: of S and dS; G: of dOut.  kWarps at a token, kBatch of its entries at a time, whose rows are asked for before any is stored to: 64 us where one after the
// other takes 77.  Others: the next stretch asked for ahead 71, rows brought to L2 ahead 73, a CTA at a token of 2048 columns 85, 24 warps an SM instead of
// 16 the same.  What bounds it is the latency of rows: DRAM is busy half of the time (4.1 TB/s), and half of what a warp's instruction takes is waiting for
// loads, with 14 warps an SM (95 registers allow two CTAs) that store between them.
template <typename T, typename G, bool kVector, int kWarps>
__global__ void __launch_bounds__(kRowsThreads, kGradCtas) ExpertsCombineGradKernel(const RowsArgs a)
{
    constexpr int kBatch = 4;
    __shared__ float sDot[2][kRowsWarps][kBatch];
    b200sp::WaitForPrevious();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, end = __ldg(a.offsets + a.experts);
    const int within = warp % kWarps;
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    constexpr int kTokens = kRowsWarps / kWarps;
    const long long step = (long long)gridDim.x * kTokens;
    long long t = (long long)blockIdx.x * kTokens + warp / kWarps;
    int turn = 0;
    TokenEntries next;
    next.Ask(a, t, lane);
    if (!HasOrder(a)) return;
    for (; t < a.tokens; t += step) {
        TokenEntries now = next;
        next.Ask(a, t + step, lane);
        const G *const grad = static_cast<const G *>(a.perToken) + t * a.ldToken;
        for (int e0 = now.range.x; e0 < now.range.y; e0 += kBatch) {
            const int first = (e0 - now.range.x) & 31, many = min(kBatch, now.range.y - e0);
            if (first == 0 && e0 > now.range.x) now.Rows(a, e0, lane);
            int place[kBatch];
            float weight[kBatch], dot[kBatch] = {};
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                place[j] = __shfl_sync(0xffffffffu, now.place, first + j);
                weight[j] = alpha * __shfl_sync(0xffffffffu, now.weight, first + j);
            }
            for (int c0 = within * kStretch; c0 < a.width; c0 += kWarps * kStretch) {
                Raw<G> raw;
                raw.template Load<kVector>(grad, c0, lane, a.width);
                Raw<T> rows[kBatch];
                if (a.dValues != nullptr) {
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        if (j < many && place[j] < end)
                            rows[j].template Load<kVector>(RowAt(static_cast<const T *>(a.perEntry), place[j], a.ldEntry), c0, lane, a.width);
                        else rows[j].Zero();
                    }
                }
                float g[8];
                raw.Floats(g);
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    if (j >= many) break;
                    if (a.dValues != nullptr && place[j] < end) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) dot[j] = fmaf(g[i], rows[j].At(i), dot[j]);
                    }
                    T *const to = RowAt(static_cast<T *>(a.out), place[j], a.ldOut);
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = place[j] < end ? weight[j] * g[i] : 0.0f;
                    Raw<T> out;
                    if (beta != 0.0f) {
                        out.template Load<kVector>(to, c0, lane, a.width);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = fmaf(beta, out.At(i), v[i]);
                    }
                    out.Set(v);
                    out.template Store<kVector>(to, c0, lane, a.width);
                }
            }
            if (a.dValues == nullptr) continue;
            float total = 0.0f;  // of entry e0 + lane
            bool in = false;     // it has an expert
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
                if (lane == j) total = dot[j], in = place[j] < end;
            }
            if constexpr (kWarps > 1) {  // a CTA's warps are all at one token; two places in turn, as others may still read the one
                if (lane < kBatch) sDot[turn][warp][lane] = total;
                __syncthreads();
                total = 0.0f;
                if (lane < kBatch)
                    for (int w = 0; w < kWarps; ++w) total += sDot[turn][warp - within + w][lane];
                turn ^= 1;
            }
            if (within == 0 && lane < many) {
                const float old = beta != 0.0f ? ValueAt(a.dValues, a.dValuesType, e0 + lane) : 0.0f;
                const float term = in ? alpha * total : 0.0f;  // whatever alpha is
                SetValue(a.dValues, a.dValuesType, e0 + lane, beta != 0.0f ? fmaf(beta, old, term) : term);
            }
        }
    }
}

// Rows in 8 bits: of tokens (kOrdered false), or every token's into the rows of its entries.  kWarps at a row, which they keep, every thread
// what it has read, in shared memory up to 1024 elements a warp, and read again beyond.  (Kept in registers, the loop unrolled around them, it took 128 of them
// and twice as long.)  What bounds it are the steps of a row, one after the other, and 130 instructions for 256 elements: 8192 rows of 4096 bf16 24 us (15 at the copy rate), of 1024 f32 11 (6.4).
template <typename T, bool kVector, int kWarps, bool kOrdered>
__global__ void __launch_bounds__(kRowsThreads, kQuantiseCtas<T>) QuantiseKernel(const RowsArgs a)
{
    constexpr int kHeld = 4;
    constexpr int kStep = kWarps * kStretch, kTokens = kRowsWarps / kWarps;
    __shared__ uint32_t sTop[2][kRowsWarps];
    __shared__ Raw<T> sHeld[kHeld][kRowsThreads];
    if (gridDim.x <= kFewCtas && a.width <= kHeld * kStep && (!kOrdered || (long long)a.nnz * max((a.width + kStretch - 1) / kStretch, kRowsWarps) <= kFewPieces))
        b200sp::LetNextStart();
    b200sp::WaitForPrevious();
    if (kOrdered && !HasOrder(a)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, within = warp % kWarps, c = within * kStretch;
    const int end = kOrdered ? __ldg(a.offsets + a.experts) : 0;
    int turn = 0;
    for (long long t = (long long)blockIdx.x * kTokens + warp / kWarps; t < a.tokens; t += (long long)gridDim.x * kTokens, turn ^= 1) {
        const T *const row = static_cast<const T *>(a.perToken) + t * a.ldToken;
        int2 entries = make_int2(0, 1);
        int mine = 0;  // where the row of entry `lane` goes
        if constexpr (kOrdered) {
            entries = EntriesOf(a, t);
            if (entries.x + lane < entries.y) mine = __ldg(a.places + entries.x + lane);
        }
        Raw<T> held[kHeld];
#pragma unroll
        for (int h = 0; h < kHeld; ++h) held[h].template Load<kVector>(row, c + h * kStep, lane, a.width);
        uint32_t top = 0;
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
            top = held[h].Top(top);
            sHeld[h][threadIdx.x] = held[h];
        }
        for (long long c0 = c + (long long)kHeld * kStep; c0 < a.width; c0 += kStep) {
            Raw<T> more;
            more.template Load<kVector>(row, (int)c0, lane, a.width);
            top = more.Top(top);
        }
        top = __reduce_max_sync(0xffffffffu, Raw<T>::TopOf(top));
        if constexpr (kWarps > 1) {  // two places in turn: one is written while others may still read the other
            if (lane == 0) sTop[turn][warp] = top;
            __syncwarp();
            asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / kWarps), "n"(32 * kWarps) : "memory");
            top = __reduce_max_sync(0xffffffffu, lane < kWarps ? sTop[turn][warp - within + lane] : 0u);
        }
        const EightBits<T> eight(top);
        for (int e0 = entries.x; e0 < entries.y; e0 += 32) {
            const int many = min(32, entries.y - e0);
            if (kOrdered && e0 > entries.x) mine = lane < many ? __ldg(a.places + e0 + lane) : 0;
            long long c0 = c;
#pragma unroll 1
            for (int h = 0; c0 < a.width; ++h, c0 += kStep) {
                Raw<T> raw;
                if (h < kHeld) raw = sHeld[h][threadIdx.x];
                else raw.template Load<kVector>(row, (int)c0, lane, a.width);
                float v[8];
                raw.Floats(v);
                const uint2 words = eight.Of(v);
                if constexpr (kOrdered) {
                    for (int j = 0; j < many; ++j) {
                        const int place = __shfl_sync(0xffffffffu, mine, j);
                        StoreBytes<kVector>(RowAt(static_cast<int8_t *>(a.out), place, a.ldOut), (int)c0, lane, a.width, place < end ? words : make_uint2(0, 0));
                    }
                } else {
                    StoreBytes<kVector>(static_cast<int8_t *>(a.out) + t * a.ldOut, (int)c0, lane, a.width, words);
                }
            }
            if (within == 0) {
                if (!kOrdered && lane == 0) a.scales[t] = eight.Scale();
                if (kOrdered && lane < many) a.scales[mine] = mine < end ? eight.Scale() : 0.0f;
            }
        }
    }
}

// ---------------------------------------------------------------- host

inline RowsArgs RowsOf(const aclsparseSpMatDescr *R, const void *buffer, uint64_t number)
{
    const PlanLayout L = PlanLayoutFor(R->nnz, R->cols);
    const char *const p = BufferStart(buffer);
    RowsArgs a{};
    a.header = reinterpret_cast<const int4 *>(p);
    a.mark = HeaderOf(R->nnz, R->cols, R->rows);
    a.number = number;
    a.offsets = reinterpret_cast<const int *>(p + L.offsets);
    a.places = reinterpret_cast<const int *>(p + L.places);
    a.rowPtr = static_cast<const int *>(R->offsets);
    a.tokens = R->rows;
    a.nnz = (int)R->nnz;
    a.experts = (int)R->cols;
    return a;
}
// CTAs for so many warps' work: as many as there are, or as many as the SMs hold.  (Twice to eight times as many: combine 57 -> 57 to 63 us, dispatch without
// its order 58 -> 58 to 62.  Rounding to 8 bits, which waits for a row before it begins with the next, gains by four times as many: 27 -> 24.)
inline unsigned RowsBlocks(long long warps, int ctas)
{
    return (unsigned)std::min<long long>((warps + kRowsWarps - 1) / kRowsWarps, (long long)b200sp_sm_count() * ctas);
}
// Calls f with types of elements; two unlike types of 16 bits are refused before.
template <typename First, typename F> cudaError_t WithSecond(First x, aclDataType second, F &&f)
{
    return WithType(second, [&](auto y) {
        if constexpr (sizeof(First) == 4 || sizeof(y) == 4 || std::is_same_v<First, decltype(y)>) return f(x, y);
        else return cudaErrorInvalidValue;
    });
}
template <typename F> cudaError_t WithTypes(aclDataType first, aclDataType second, F &&f)
{
    return WithType(first, [&](auto x) { return WithSecond(x, second, f); });
}
inline bool UnlikeHalves(aclDataType x, aclDataType y) { return x != ACL_FLOAT && y != ACL_FLOAT && x != y; }

// An output of numbers of one type, `size` of them.
inline aclsparseStatus_t CheckNumbers(const aclsparseDnVecDescr *v, int64_t size, aclDataType type, int bytes)
{
    if (v == nullptr || v->magic != b200sp::kDnVecMagic) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (v->valueType != type) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (v->size != size || v->values == nullptr || !OnBoundary(v->values, bytes)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}
inline aclsparseStatus_t CheckStarts(const aclsparseSpMatDescr *R, const aclsparseDnVecDescr *offsets)
{
    return offsets == nullptr ? ACL_SPARSE_STATUS_SUCCESS : CheckNumbers(offsets, R->cols + 1, ACL_INT32, 4);
}
inline aclsparseStatus_t CheckWeights(const aclsparseSpMatDescr *R)
{
    if (!IsFloatType(R->valueType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->values == nullptr || !OnBoundary(R->values, BytesOf(R->valueType))) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}
// Rows of 8 bits.
inline aclsparseStatus_t CheckBytes(const aclsparseDnMatDescr *m)
{
    if (m == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (m->order != ACL_SPARSE_ORDER_ROW || m->valueType != ACL_INT8) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (m->rows > INT32_MAX || m->cols > kMostCounted || m->ld > INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    return m->values == nullptr ? ACL_SPARSE_STATUS_INVALID_VALUE : ACL_SPARSE_STATUS_SUCCESS;
}

template <typename T, bool kOrdered, int kWarps> cudaError_t LaunchQuantise(const RowsArgs &a, bool vectors, cudaStream_t stream)
{
    b200sp_note_launches(1);
    const unsigned blocks = RowsBlocks(a.tokens * kWarps, kQuantiseCtas<T> * 4);
    return vectors ? b200sp::LaunchChained(QuantiseKernel<T, true, kWarps, kOrdered>, blocks, kRowsThreads, 0, stream, a)
                   : b200sp::LaunchChained(QuantiseKernel<T, false, kWarps, kOrdered>, blocks, kRowsThreads, 0, stream, a);
}
// As many warps as keep a row in shared memory, 1024 elements each; where there are few rows, a CTA's.
template <typename T, bool kOrdered> cudaError_t LaunchQuantise(const RowsArgs &a, bool vectors, cudaStream_t stream)
{
    if (a.width > 4096 || a.tokens < (long long)b200sp_sm_count() * 4) return LaunchQuantise<T, kOrdered, 8>(a, vectors, stream);
    if (a.width > 2048) return LaunchQuantise<T, kOrdered, 4>(a, vectors, stream);
    if (a.width > 1024) return LaunchQuantise<T, kOrdered, 2>(a, vectors, stream);
    return LaunchQuantise<T, kOrdered, 1>(a, vectors, stream);
}
inline bool QuantiseVectors(const aclsparseDnMatDescr *X, const aclsparseDnMatDescr *Q)
{
    return RowsAligned(X) && OnBoundary(Q->values, 8) && Q->ld % 8 == 0;
}
