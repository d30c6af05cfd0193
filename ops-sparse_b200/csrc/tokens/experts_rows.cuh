// Rows of tokens in the order of their experts, and back: included by experts.cu.
//
// dispatch: S[place(i)] = alpha X[token(i)]; combine: out[t] = alpha sum of w_i S[place(i)]; its gradient: dS[place(i)] = alpha w_i dOut[t],
// dw_i = alpha <dOut[t], S[place(i)]>.  All go by tokens, whose entries lie side by side in R: a token's row is read (or written) once and stays in
// registers while the rows of its entries, which lie anywhere, are written (or read).  What bounds them is DRAM.
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

constexpr int kRowsThreads = 256, kRowsWarps = kRowsThreads / 32;

// What every call of this file begins with: false without an order.
__device__ __forceinline__ bool RowsBegin(const RowsArgs &a)
{
    b200sp::WaitForPrevious();
    if (!StartsWith(a.header, a.mark, a.number)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicMax(&gExpertsError, kNoOrder);
        return false;
    }
    if (a.starts != nullptr && blockIdx.x == 0)
        for (int e = threadIdx.x; e <= a.experts; e += kRowsThreads) a.starts[e] = __ldg(a.offsets + e);
    return true;
}
// The entries of a token, whatever the offsets say.
__device__ __forceinline__ int2 EntriesOf(const RowsArgs &a, long long token)
{
    return make_int2(max(0, __ldg(a.rowPtr + token)), min(a.nnz, __ldg(a.rowPtr + token + 1)));
}

template <typename In, typename Out> constexpr int kStretch = 16 / (sizeof(In) < sizeof(Out) ? (int)sizeof(In) : (int)sizeof(Out));

template <typename In, typename Out, bool kVector> __global__ void __launch_bounds__(kRowsThreads) ExpertsDispatchKernel(const RowsArgs a)
{
    constexpr int kN = kStretch<In, Out>;
    if (!RowsBegin(a)) return;
    const int lane = threadIdx.x & 31, end = __ldg(a.offsets + a.experts);
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    Units u((long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5), (long long)gridDim.x * kRowsWarps, (a.width + 32 * kN - 1) / (32 * kN));
    for (; u.row < a.tokens; u.Next()) {
        const int2 entries = EntriesOf(a, u.row);
        const int c0 = u.stretch * 32 * kN;
        float v[kN];
        LoadStretch<In, kN, kVector>(static_cast<const In *>(a.perToken) + u.row * a.ldToken, c0, lane, a.width, v);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] *= alpha;
        for (int e0 = entries.x; e0 < entries.y; e0 += 32) {
            const int mine = e0 + lane < entries.y ? __ldg(a.places + e0 + lane) : 0, many = min(32, entries.y - e0);
            for (int j = 0; j < many; ++j) {
                const int place = __shfl_sync(0xffffffffu, mine, j);
                Out *const to = static_cast<Out *>(a.out) + place * a.ldOut;
                float w[kN];
                if (beta != 0.0f) LoadStretch<Out, kN, kVector>(to, c0, lane, a.width, w);
#pragma unroll
                for (int i = 0; i < kN; ++i) {
                    const float x = place < end ? v[i] : 0.0f;
                    w[i] = beta != 0.0f ? fmaf(beta, w[i], x) : x;
                }
                StoreStretch<Out, kN, kVector>(to, c0, lane, a.width, w);
            }
        }
    }
}

template <typename In, typename Out, bool kVector> __global__ void __launch_bounds__(kRowsThreads) ExpertsCombineKernel(const RowsArgs a)
{
    constexpr int kN = kStretch<In, Out>;
    if (!RowsBegin(a)) return;
    const int lane = threadIdx.x & 31, end = __ldg(a.offsets + a.experts);
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    Units u((long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5), (long long)gridDim.x * kRowsWarps, (a.width + 32 * kN - 1) / (32 * kN));
    for (; u.row < a.tokens; u.Next()) {
        const int2 entries = EntriesOf(a, u.row);
        const int c0 = u.stretch * 32 * kN;
        float sum[kN] = {};
        for (int e0 = entries.x; e0 < entries.y; e0 += 32) {
            int mine = end;
            float weight = 1.0f;
            if (e0 + lane < entries.y) {
                mine = __ldg(a.places + e0 + lane);
                if (a.weights != nullptr) weight = ValueAt(a.weights, a.weightType, e0 + lane);
            }
            const int many = min(32, entries.y - e0);
            for (int j = 0; j < many; ++j) {
                const int place = __shfl_sync(0xffffffffu, mine, j);
                const float w = __shfl_sync(0xffffffffu, weight, j);
                if (place >= end) continue;
                float v[kN];
                LoadStretch<In, kN, kVector>(static_cast<const In *>(a.perEntry) + place * a.ldEntry, c0, lane, a.width, v);
#pragma unroll
                for (int i = 0; i < kN; ++i) sum[i] = fmaf(w, v[i], sum[i]);
            }
        }
        Out *const to = static_cast<Out *>(a.out) + u.row * a.ldOut;
        float old[kN];
        if (beta != 0.0f) LoadStretch<Out, kN, kVector>(to, c0, lane, a.width, old);
#pragma unroll
        for (int i = 0; i < kN; ++i) sum[i] = beta != 0.0f ? fmaf(beta, old[i], alpha * sum[i]) : alpha * sum[i];
        StoreStretch<Out, kN, kVector>(to, c0, lane, a.width, sum);
    }
}

// T: of S and dS; G: of dOut.  kWarps at a token, eight of its entries at a time.
template <typename T, typename G, bool kVector, int kWarps>
__global__ void __launch_bounds__(kRowsThreads) ExpertsCombineGradKernel(const RowsArgs a)
{
    constexpr int kN = kStretch<T, G>, kBatch = 8;
    __shared__ float sDot[kRowsWarps][kBatch];
    if (!RowsBegin(a)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, end = __ldg(a.offsets + a.experts);
    const int within = warp % kWarps;
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    constexpr int kTokens = kRowsWarps / kWarps;
    for (long long t = (long long)blockIdx.x * kTokens + warp / kWarps; t < a.tokens; t += (long long)gridDim.x * kTokens) {
        const int2 entries = EntriesOf(a, t);
        const G *const grad = static_cast<const G *>(a.perToken) + t * a.ldToken;
        for (int e0 = entries.x; e0 < entries.y; e0 += kBatch) {
            int mine = 0;
            float weight = 0.0f;
            const int many = min(kBatch, entries.y - e0);
            if (lane < many) {
                mine = __ldg(a.places + e0 + lane);
                weight = alpha * ValueAt(a.weights, a.weightType, e0 + lane);
            }
            float dot[kBatch] = {};
            for (int c0 = within * 32 * kN; c0 < a.width; c0 += kWarps * 32 * kN) {
                float g[kN];
                LoadStretch<G, kN, kVector>(grad, c0, lane, a.width, g);
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    if (j >= many) break;
                    const int place = __shfl_sync(0xffffffffu, mine, j);
                    const float w = __shfl_sync(0xffffffffu, weight, j);
                    float v[kN];
                    if (a.dValues != nullptr && place < end) {
                        LoadStretch<T, kN, kVector>(static_cast<const T *>(a.perEntry) + place * a.ldEntry, c0, lane, a.width, v);
#pragma unroll
                        for (int i = 0; i < kN; ++i) dot[j] = fmaf(g[i], v[i], dot[j]);
                    }
                    T *const to = static_cast<T *>(a.out) + place * a.ldOut;
                    if (beta != 0.0f) LoadStretch<T, kN, kVector>(to, c0, lane, a.width, v);
#pragma unroll
                    for (int i = 0; i < kN; ++i) {
                        const float x = place < end ? w * g[i] : 0.0f;
                        v[i] = beta != 0.0f ? fmaf(beta, v[i], x) : x;
                    }
                    StoreStretch<T, kN, kVector>(to, c0, lane, a.width, v);
                }
            }
            if (a.dValues == nullptr) continue;
            float total = 0.0f;  // of entry `lane`
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
                if (lane == j) total = dot[j];
            }
            if constexpr (kWarps > 1) {
                if (lane < kBatch) sDot[warp][lane] = total;
                __syncthreads();
                total = 0.0f;
                if (lane < kBatch)
                    for (int w = 0; w < kWarps; ++w) total += sDot[warp - within + w][lane];
                __syncthreads();  // a CTA's warps are all at one token
            }
            if (within == 0 && lane < many) {
                const float old = beta != 0.0f ? beta * ValueAt(a.dValues, a.dValuesType, e0 + lane) : 0.0f;
                SetValue(a.dValues, a.dValuesType, e0 + lane, beta != 0.0f ? fmaf(alpha, total, old) : alpha * total);
            }
        }
    }
}

// Rows in 8 bits: of tokens (kOrdered false), or every token's into the rows of its entries.  kWarps at a row, which they keep in registers
// up to kHeld elements a thread and read again beyond.
template <typename T, bool kVector, int kWarps, bool kOrdered>
__global__ void __launch_bounds__(kRowsThreads) QuantiseKernel(const RowsArgs a)
{
    constexpr int kN = 8, kHeld = 32 * 4 / (kN * (int)sizeof(T));  // stretches: 32 registers
    constexpr int kStep = kWarps * 32 * kN, kTokens = kRowsWarps / kWarps;
    __shared__ uint32_t sTop[kRowsWarps];
    if constexpr (kOrdered) {
        if (!RowsBegin(a)) return;
    } else {
        b200sp::WaitForPrevious();
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, within = warp % kWarps;
    const int end = kOrdered ? __ldg(a.offsets + a.experts) : 0;
    for (long long t = (long long)blockIdx.x * kTokens + warp / kWarps; t < a.tokens; t += (long long)gridDim.x * kTokens) {
        const T *const row = static_cast<const T *>(a.perToken) + t * a.ldToken;
        const int2 entries = kOrdered ? EntriesOf(a, t) : make_int2(0, 1);
        const int c = within * 32 * kN;
        T held[kHeld][kN];
        uint32_t top = 0;
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
            if (c + h * kStep >= a.width) break;
            float v[kN];
            LoadStretch<T, kN, kVector>(row, c + h * kStep, lane, a.width, v);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                held[h][i] = FromFloat<T>(v[i]);
                top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
            }
        }
        for (long long c0 = c + (long long)kHeld * kStep; c0 < a.width; c0 += kStep) {
            float v[kN];
            LoadStretch<T, kN, kVector>(row, (int)c0, lane, a.width, v);
#pragma unroll
            for (int i = 0; i < kN; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if constexpr (kWarps > 1) {
            if (lane == 0) sTop[warp] = top;
            __syncthreads();
            top = __reduce_max_sync(0xffffffffu, lane < kWarps ? sTop[warp - within + lane] : 0u);
            __syncthreads();  // a CTA's warps are all at one row
        }
        const EightBits eight(top);
        auto store = [&](int8_t *to, int c0, const int (&q)[kN]) {
            if constexpr (kVector) {
                const int at = c0 + lane * kN;
                if (at + kN <= a.width) {
                    uint2 words;
                    words.x = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | q[3] << 24;
                    words.y = (q[4] & 255) | (q[5] & 255) << 8 | (q[6] & 255) << 16 | q[7] << 24;
                    *reinterpret_cast<uint2 *>(to + at) = words;
                } else {
#pragma unroll
                    for (int i = 0; i < kN; ++i)
                        if (at + i < a.width) to[at + i] = (int8_t)q[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < kN; ++i)
                    if (c0 + 32 * i + lane < a.width) to[c0 + 32 * i + lane] = (int8_t)q[i];
            }
        };
        for (int e0 = entries.x; e0 < entries.y; e0 += 32) {
            const int many = min(32, entries.y - e0);
            int mine = 0;
            if (kOrdered && lane < many) mine = __ldg(a.places + e0 + lane);
            auto write = [&](int c0, const float (&v)[kN]) {
                int q[kN], zeros[kN] = {};
#pragma unroll
                for (int i = 0; i < kN; ++i) q[i] = eight.Of(v[i]);
                if constexpr (kOrdered) {
                    for (int j = 0; j < many; ++j) {
                        const int place = __shfl_sync(0xffffffffu, mine, j);
                        int8_t *const to = static_cast<int8_t *>(a.out) + place * a.ldOut;
                        if (place < end) store(to, c0, q);
                        else store(to, c0, zeros);
                    }
                } else {
                    store(static_cast<int8_t *>(a.out) + t * a.ldOut, c0, q);
                }
            };
#pragma unroll
            for (int h = 0; h < kHeld; ++h) {
                if (c + h * kStep >= a.width) break;
                float v[kN];
#pragma unroll
                for (int i = 0; i < kN; ++i) v[i] = ToFloat(held[h][i]);
                write(c + h * kStep, v);
            }
            for (long long c0 = c + (long long)kHeld * kStep; c0 < a.width; c0 += kStep) {
                float v[kN];
                LoadStretch<T, kN, kVector>(row, (int)c0, lane, a.width, v);
                write((int)c0, v);
            }
            if (within == 0) {
                if (!kOrdered && lane == 0) a.scales[t] = eight.scale;
                if (kOrdered && lane < many) a.scales[mine] = mine < end ? eight.scale : 0.0f;
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
// CTAs for so many warps' work: as many as there are, or eight to an SM.
inline unsigned RowsBlocks(long long warps)
{
    return (unsigned)std::min<long long>((warps + kRowsWarps - 1) / kRowsWarps, (long long)b200sp_sm_count() * 8);
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

template <typename T, bool kOrdered> cudaError_t LaunchQuantise(const RowsArgs &a, bool vectors, cudaStream_t stream)
{
    // A warp for a row, as long as it keeps the row in registers and there are rows for all SMs; else a CTA.
    const bool cta = a.width > 32 * 128 / (int)sizeof(T) || a.tokens < (long long)b200sp_sm_count() * kRowsWarps;
    const unsigned blocks = RowsBlocks(cta ? a.tokens * kRowsWarps : a.tokens);
    b200sp_note_launches(1);
    if (cta)
        return vectors ? b200sp::LaunchChained(QuantiseKernel<T, true, kRowsWarps, kOrdered>, blocks, kRowsThreads, 0, stream, a)
                       : b200sp::LaunchChained(QuantiseKernel<T, false, kRowsWarps, kOrdered>, blocks, kRowsThreads, 0, stream, a);
    return vectors ? b200sp::LaunchChained(QuantiseKernel<T, true, 1, kOrdered>, blocks, kRowsThreads, 0, stream, a)
                   : b200sp::LaunchChained(QuantiseKernel<T, false, 1, kOrdered>, blocks, kRowsThreads, 0, stream, a);
}
inline bool QuantiseVectors(const aclsparseDnMatDescr *X, const aclsparseDnMatDescr *Q)
{
    return RowsAligned(X) && OnBoundary(Q->values, 8) && Q->ld % 8 == 0;
}
