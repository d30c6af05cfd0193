// b200spRoute, b200spRouteGrad: the k best experts of every token as a CSR matrix, and the gradient of its values.
//
// A warp has a token; its lanes hold the token's logits, 1 to 32 each (expert 32 j + lane).  The k experts are taken one after the
// other: the largest key of the warp, then the lowest expert that has it.  Keys are the selection values as unsigned
// integers of the same order.
// The choice is that of exact arithmetic.  Without a bias it is made on the logits themselves, which both scores ascend
// with.  With one, p + bias is computed in f32 together with a bound of its error; where another expert lies as near the last
// one taken as the two bounds together, or a group that is kept as near one that is not, the row is done again in
// f64.  Of 16,384 rows of 256 experts some ten are.
#include <cmath>

#include "b200sp_tokens.h"
#include "tokens/common.cuh"

namespace {

using namespace b200sp_tokens;

constexpr int kMaxExperts = 1024, kMaxChosen = 32, kMaxGroups = 32;
template <int kPer> constexpr int kRouteWarps = kPer < 32 ? 4 : 2;  // of a CTA: what shared memory has room for
constexpr unsigned kAll = 0xffffffffu;

struct RouteArgs {
    const void *logits;
    const float *bias;
    long long ld;
    int tokens, experts, k;
    int sigmoid, groups, kept, top2, renormalise;
    float scale;
    int *offsets, *columns;
    void *values;
};

template <typename Real> struct Limits;
template <> struct Limits<float> {
    static __device__ __forceinline__ float Lowest() { return -INFINITY; }
};
template <> struct Limits<double> {
    static __device__ __forceinline__ double Lowest() { return -(double)INFINITY; }
};

__device__ __forceinline__ float Exp(float v) { return expf(v); }
__device__ __forceinline__ double Exp(double v) { return exp(v); }

template <typename Real> __device__ __forceinline__ Real WarpMax(Real v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const Real o = __shfl_xor_sync(kAll, v, d);
        v = o > v ? o : v;
    }
    return v;
}
template <typename Real> __device__ __forceinline__ Real WarpSum(Real v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
    return v;
}

// Numbers of the same order as the values (no NaN among them); 0 is below all of them.
__device__ __forceinline__ uint32_t KeyOf(float v)
{
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long KeyOf(double v)
{
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint32_t MaxKey(uint32_t v) { return __reduce_max_sync(kAll, v); }
__device__ __forceinline__ unsigned long long MaxKey(unsigned long long v)
{
    const uint32_t high = __reduce_max_sync(kAll, (uint32_t)(v >> 32));
    const uint32_t low = __reduce_max_sync(kAll, (uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
    return (unsigned long long)high << 32 | low;
}

// Scores of the lanes' logits (masked: -infinity), 0 for the masked.
template <typename Real, int kPer> __device__ __forceinline__ void Scores(const RouteArgs &a, const float (&x)[kPer], Real (&p)[kPer], float *most)
{
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) p[j] = (Real)1 / ((Real)1 + Exp(-(Real)x[j]));
        *most = 0.0f;
        return;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; ++j) m = fmaxf(m, x[j]);
    m = WarpMax(m);
    Real sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        // infinite logits share the score
        p[j] = x[j] == -INFINITY ? (Real)0 : x[j] == m ? (Real)1 : Exp((Real)x[j] - (Real)m);
        sum += p[j];
    }
    sum = WarpSum(sum);
    const Real inv = sum > 0 ? (Real)1 / sum : (Real)0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) p[j] *= inv;
    *most = m;
}

// How far p, in f32, may be from the score: expf 2 units of its last place and the division 1, a softmax's sum of kPer + 5 additions and the
// difference of its logits, each 2^-24 of p (a few more are allowed).
__device__ __forceinline__ float ErrorOf(const RouteArgs &a, float x, float p, float most)
{
    constexpr float kUnit = 6.0e-8f;
    return p * (a.sigmoid ? 8 * kUnit : kUnit * (64.0f + 2.0f * fminf(most - x, 200.0f)));
}

struct Chosen {
    uint32_t mine;       // bit j: the lane's expert 32 j + lane is taken
    uint32_t weightless; // and has no selection value
    bool unsure;         // f32 does not tell
};

template <typename Real, int kPer>
__device__ __forceinline__ Chosen Choose(const RouteArgs &a, const float (&x)[kPer], const Real (&p)[kPer], float most, float *sRow, int lane)
{
    constexpr bool kBounds = sizeof(Real) == 4;
    Chosen c{0, 0, false};
    Real s[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int e = 32 * j + lane;
        s[j] = (Real)x[j];
        if (a.bias != nullptr && e < a.experts) {
            const float b = __ldg(a.bias + e);
            s[j] = x[j] == -INFINITY || !(b > -INFINITY) ? Limits<Real>::Lowest() : p[j] + (Real)b;
        }
    }
    if (a.groups > 1) {
        // Lanes side by side on a group: the two best of their experts, then of the group.
        Real *const sValues = reinterpret_cast<Real *>(sRow);
        const bool sums = a.top2 != 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = 32 * j + lane;
            const Real v = sums && a.bias == nullptr ? (x[j] == -INFINITY ? Limits<Real>::Lowest() : p[j]) : s[j];
            if (e < a.experts) sValues[e + (e >> 5)] = v;
        }
        __syncwarp();
        int wide = 32;  // lanes of a group
        while (wide * a.groups > 32) wide >>= 1;
        const int group = lane / wide, size = a.experts / a.groups;
        Real first = Limits<Real>::Lowest(), second = Limits<Real>::Lowest();
        if (group < a.groups) {
            for (int i = lane % wide; i < size; i += wide) {
                const int e = group * size + i;
                const Real v = sValues[e + (e >> 5)];
                if (v > first) {
                    second = first;
                    first = v;
                } else if (v > second) {
                    second = v;
                }
            }
        }
        for (int d = 1; d < wide; d <<= 1) {
            const Real f = __shfl_xor_sync(kAll, first, d), t = __shfl_xor_sync(kAll, second, d);
            const Real low = f > first ? first : f;
            if (f > first) first = f;
            Real high = t > second ? t : second;
            second = low > high ? low : high;
        }
        __syncwarp();
        const Real value = sums && second > Limits<Real>::Lowest() ? first + second : first;
        // lane g < groups: group g
        const Real mine = __shfl_sync(kAll, value, (lane * wide) & 31);
        int place = 0;
        for (int g = 0; g < a.groups; ++g) {
            const Real o = __shfl_sync(kAll, mine, g);
            place += o > mine || (o == mine && g < lane);
        }
        const unsigned open = __ballot_sync(kAll, lane < a.groups && place < a.kept);
        if (kBounds && (a.bias != nullptr || sums)) {
            // both values of a sum have an error of at most ErrorOf(p = 1), each addition half a unit of its result
            const float unit = a.sigmoid ? 2.0e-6f : 1.5e-5f;
            for (int g = 0; g < a.groups; ++g) {
                const float o = (float)__shfl_sync(kAll, mine, g), own = (float)mine;
                const bool apart = lane < a.groups && (((open >> g) ^ (open >> lane)) & 1) != 0;
                c.unsure |= apart && fabsf(o - own) <= unit + 2.4e-7f * (fabsf(o) + fabsf(own));
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = 32 * j + lane;
            if (e < a.experts && !(open >> (e / size) & 1)) s[j] = Limits<Real>::Lowest();
        }
    }
    using Key = decltype(KeyOf(Real{}));
    Key key[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) key[j] = 32 * j + lane < a.experts ? KeyOf(s[j]) : 0;
    const Key nothing = KeyOf(Limits<Real>::Lowest());
    Real lastValue = 0;
    float lastX = 0, lastBias = 0, lastError = 0;
    for (int i = 0; i < a.k; ++i) {
        Key best = 0;
        int at = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (key[j] > best) {
                best = key[j];
                at = j;
            }
        }
        const Key top = MaxKey(best);
        const unsigned e = __reduce_min_sync(kAll, best == top && top != 0 ? 32u * at + lane : ~0u);
        const bool won = (e & 31) == (unsigned)lane && e != ~0u;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (!won || (int)(e >> 5) != j) continue;
            key[j] = 0;
            c.mine |= 1u << j;
            if (top == nothing) c.weightless |= 1u << j;
            if (kBounds && i == a.k - 1) {
                lastValue = s[j];
                lastX = x[j];
                lastError = ErrorOf(a, x[j], (float)p[j], most);
                lastBias = a.bias != nullptr ? __ldg(a.bias + e) : 0.0f;
            }
        }
        if (kBounds && i == a.k - 1 && a.bias != nullptr) {
            const int from = (int)(e & 31);
            lastValue = __shfl_sync(kAll, lastValue, from);
            lastX = __shfl_sync(kAll, lastX, from);
            lastError = __shfl_sync(kAll, lastError, from);
            lastBias = __shfl_sync(kAll, lastBias, from);
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                // Neighbours of the last one taken, but for those that are its equals in exact arithmetic too.
                if (32 * j + lane >= a.experts || 32u * j + lane == e || key[j] == nothing) continue;
                const float gap = fabsf((float)(s[j] - lastValue));
                const float room = ErrorOf(a, x[j], (float)p[j], most) + lastError + 1.2e-7f * (fabsf((float)s[j]) + fabsf((float)lastValue));
                if (gap <= room) c.unsure |= !(x[j] == lastX && __ldg(a.bias + 32 * j + lane) == lastBias);
            }
        }
    }
    c.unsure = kBounds && __any_sync(kAll, c.unsure);
    return c;
}

template <int kPer> __device__ __noinline__ Chosen ChooseExactly(const RouteArgs &a, const float *sLogits, float *sRow, int lane)
{
    float x[kPer], most;
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = sLogits[32 * j + lane];
    double p[kPer];
    Scores<double, kPer>(a, x, p, &most);
    return Choose<double, kPer>(a, x, p, most, sRow, lane);
}

template <typename In, typename Out, int kPer> __global__ void __launch_bounds__(32 * kRouteWarps<kPer>) RouteKernel(const RouteArgs a)
{
    // of a warp: its selection values by expert, a word apart every 32 (f64 too), and its logits for a second pass
    __shared__ double sRows[kRouteWarps<kPer>][33 * kPer];
    __shared__ float sLogits[kRouteWarps<kPer>][32 * kPer];
    b200sp::WaitForPrevious();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long token = (long long)blockIdx.x * kRouteWarps<kPer> + warp;
    if (token >= a.tokens) return;
    const In *const row = static_cast<const In *>(a.logits) + token * a.ld;
    float x[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        x[j] = 32 * j + lane < a.experts ? ToFloat(row[32 * j + lane]) : -INFINITY;
        if (!(x[j] > -INFINITY)) x[j] = -INFINITY;  // NaN, too
    }
    float p[kPer], most;
    Scores<float, kPer>(a, x, p, &most);
    float *const sRow = reinterpret_cast<float *>(sRows[warp]);
    Chosen c = Choose<float, kPer>(a, x, p, most, sRow, lane);
    if (c.unsure) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) sLogits[warp][32 * j + lane] = x[j];
        __syncwarp();
        c = ChooseExactly<kPer>(a, sLogits[warp], sRow, lane);
    }
    float sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (c.weightless >> j & 1) p[j] = 0.0f;
        if (c.mine >> j & 1) sum += p[j];
    }
    float by = a.scale;
    if (a.renormalise) {
        sum = WarpSum(sum);
        by = sum > 0 ? a.scale / sum : 0.0f;
    }
    long long at = token * a.k;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const unsigned taken = __ballot_sync(kAll, c.mine >> j & 1);
        if (c.mine >> j & 1) {
            const long long to = at + __popc(taken & ((1u << lane) - 1u));
            a.columns[to] = 32 * j + lane;
            static_cast<Out *>(a.values)[to] = FromFloat<Out>(p[j] * by);
        }
        at += __popc(taken);
    }
    if (lane == 0) a.offsets[token] = (int)(token * a.k);
    if (lane == 0 && token == a.tokens - 1) a.offsets[a.tokens] = (int)((token + 1) * a.k);
}

// ---------------------------------------------------------------- gradient

struct RouteGradArgs {
    const void *logits;
    long long ld, ldOut;
    int tokens, experts, k;
    int sigmoid, renormalise;
    float scale;
    const int *columns;
    const void *values, *grad;
    int valueType, gradType;
    void *out;
};

__device__ __forceinline__ float LoadAs(const void *p, long long i, int type)
{
    if (type == ACL_FLOAT16) return ToFloat(static_cast<const __half *>(p)[i]);
    if (type == ACL_BF16) return ToFloat(static_cast<const __nv_bfloat16 *>(p)[i]);
    return static_cast<const float *>(p)[i];
}

// Lane i has entry i of the token's row.  With q the weights over scale and g their gradients (times scale):
//   softmax, renormalised   dx = q (g - sum g q): the softmax of the chosen logits alone
//   sigmoid, renormalised   dx = (g - sum g q) / (sum s) * s (1 - s)
//   sigmoid                 dx = g s (1 - s)
//   softmax                 dx = p (g - sum g p) for the chosen, -p sum g p for the others
template <typename T, int kPer> __global__ void __launch_bounds__(32 * kRouteWarps<kPer>) RouteGradKernel(const RouteGradArgs a)
{
    __shared__ float sRows[kRouteWarps<kPer>][32 * kPer];
    b200sp::WaitForPrevious();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long token = (long long)blockIdx.x * kRouteWarps<kPer> + warp;
    if (token >= a.tokens) return;
    float *const sRow = sRows[warp];
    const T *const row = static_cast<const T *>(a.logits) + token * a.ld;
    int col = -1;
    float g = 0.0f, x = -INFINITY;
    if (lane < a.k) {
        const long long i = token * a.k + lane;
        col = __ldg(a.columns + i);
        if (col < 0 || col >= a.experts || LoadAs(a.values, i, a.valueType) == 0.0f) col = -1;
        if (col >= 0) {
            g = a.scale * LoadAs(a.grad, i, a.gradType);
            x = ToFloat(row[col]);
            if (!(x > -INFINITY)) col = -1, g = 0.0f, x = -INFINITY;
        }
    }
    const bool dense = !a.sigmoid && !a.renormalise;
    float dx = 0.0f;
    if (dense) {
        float v[kPer], m = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            v[j] = 32 * j + lane < a.experts ? ToFloat(row[32 * j + lane]) : -INFINITY;
            if (!(v[j] > -INFINITY)) v[j] = -INFINITY;
            m = fmaxf(m, v[j]);
        }
        m = WarpMax(m);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            v[j] = v[j] == -INFINITY ? 0.0f : v[j] == m ? 1.0f : expf(v[j] - m);
            sum += v[j];
        }
        sum = WarpSum(sum);
        const float inv = sum > 0 ? 1.0f / sum : 0.0f;
        const float p = col < 0 ? 0.0f : (x == m ? 1.0f : expf(x - m)) * inv;
        const float dot = WarpSum(g * p);
#pragma unroll
        for (int j = 0; j < kPer; ++j) sRow[32 * j + lane] = -v[j] * inv * dot;
        dx = p * (g - dot);
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) sRow[32 * j + lane] = 0.0f;
        if (a.sigmoid) {
            const float s = col < 0 ? 0.0f : 1.0f / (1.0f + expf(-x));
            const float rest = col < 0 ? 0.0f : 1.0f / (1.0f + expf(x));  // 1 - s, exactly enough where s is near 1
            if (a.renormalise) {
                const float sum = WarpSum(s), inv = sum > 0 ? 1.0f / sum : 0.0f;
                g = (g - WarpSum(g * s) * inv) * inv;
            }
            dx = g * s * rest;
        } else {
            const float m = WarpMax(x);
            const float e = col < 0 ? 0.0f : x == m ? 1.0f : expf(x - m);
            const float sum = WarpSum(e), q = sum > 0 ? e / sum : 0.0f;
            dx = q * (g - WarpSum(g * q));
        }
    }
    __syncwarp();
    if (col >= 0) sRow[col] = dx;
    __syncwarp();
    T *const out = static_cast<T *>(a.out) + token * a.ldOut;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (32 * j + lane < a.experts) out[32 * j + lane] = FromFloat<T>(sRow[32 * j + lane]);
}

// ---------------------------------------------------------------- host

// f with the logits of a lane as a constant.
template <typename F> auto WithPer(int experts, F &&f)
{
    if (experts <= 32) return f(std::integral_constant<int, 1>{});
    if (experts <= 64) return f(std::integral_constant<int, 2>{});
    if (experts <= 128) return f(std::integral_constant<int, 4>{});
    if (experts <= 256) return f(std::integral_constant<int, 8>{});
    if (experts <= 512) return f(std::integral_constant<int, 16>{});
    return f(std::integral_constant<int, 32>{});
}

template <int kPer> unsigned RouteBlocks(long long tokens) { return (unsigned)((tokens + kRouteWarps<kPer> - 1) / kRouteWarps<kPer>); }

aclsparseStatus_t CheckRoute(const b200spRouteRule *rule, const aclsparseDnMatDescr *logits, const aclsparseSpMatDescr *R)
{
    if (rule == nullptr || R == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rule->score != B200SP_ROUTE_SOFTMAX && rule->score != B200SP_ROUTE_SIGMOID) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rule->groupScore != B200SP_GROUP_MAX && rule->groupScore != B200SP_GROUP_TOP2) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rule->renormalise != 0 && rule->renormalise != 1) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (!std::isfinite(rule->scale)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rule->groups < 1 || rule->groupsKept < 1 || rule->groupsKept > rule->groups) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckDense(logits);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (R->format != ACL_SPARSE_FORMAT_CSR) return ACL_SPARSE_STATUS_MATRIX_TYPE_NOT_SUPPORTED;
    const aclsparseStatus_t idx = b200sp::CheckExecIndexTypes(R->offsetType, R->indexType);
    if (idx != ACL_SPARSE_STATUS_SUCCESS) return idx;
    if (R->base != ACL_SPARSE_INDEX_BASE_ZERO || !IsFloatType(R->valueType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (logits->rows != R->rows || logits->cols != R->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (R->cols > kMaxExperts || rule->groups > kMaxGroups) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->nnz > INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->nnz % R->rows != 0 || R->nnz == 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const int64_t k = R->nnz / R->rows;
    if (k > kMaxChosen) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->cols % rule->groups != 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (k > R->cols / rule->groups * rule->groupsKept) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (R->offsets == nullptr || R->indices == nullptr || R->values == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

}  // namespace

extern "C" {

aclsparseStatus_t b200spRoute(aclsparseHandle_t handle, const b200spRouteRule *rule, aclsparseConstDnMatDescr_t logits,
                              aclsparseConstDnVecDescr_t bias, aclsparseSpMatDescr_t matR)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    const aclsparseStatus_t st = CheckRoute(rule, logits, matR);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (bias != nullptr) {
        if (bias->magic != b200sp::kDnVecMagic || bias->size != matR->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
        if (bias->valueType != ACL_FLOAT) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    const OnDevice device(handle);
    RouteArgs a{logits->values, bias != nullptr ? static_cast<const float *>(bias->values) : nullptr, logits->ld, (int)matR->rows,
                (int)matR->cols, (int)(matR->nnz / matR->rows), rule->score == B200SP_ROUTE_SIGMOID, rule->groups, rule->groupsKept,
                rule->groupScore == B200SP_GROUP_TOP2, rule->renormalise, rule->scale, static_cast<int *>(matR->offsets),
                static_cast<int *>(matR->indices), matR->values};
    if (a.kept == a.groups) a.groups = a.kept = 1;  // all are kept
    const cudaError_t e = WithPer(a.experts, [&](auto per) {
        return WithType(logits->valueType, [&](auto in) {
            return WithType(matR->valueType, [&](auto out) {
                constexpr int kPer = decltype(per)::value;
                b200sp_note_launches(1);
                return b200sp::LaunchChained(RouteKernel<decltype(in), decltype(out), kPer>, RouteBlocks<kPer>(a.tokens),
                                             32 * kRouteWarps<kPer>, 0, handle->stream, a);
            });
        });
    });
    return Finished(e, "b200spRoute");
}

aclsparseStatus_t b200spRouteGrad(aclsparseHandle_t handle, const b200spRouteRule *rule, aclsparseConstDnMatDescr_t logits,
                                  aclsparseConstSpMatDescr_t matR, aclsparseConstDnVecDescr_t dValues,
                                  aclsparseDnMatDescr_t dLogits)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    aclsparseStatus_t st = CheckRoute(rule, logits, matR);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckDense(dLogits);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (dValues == nullptr || dValues->magic != b200sp::kDnVecMagic) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (!IsFloatType(dValues->valueType) || dLogits->valueType != logits->valueType) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (dValues->size != matR->nnz || dLogits->rows != logits->rows || dLogits->cols != logits->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    const RouteGradArgs a{logits->values, logits->ld, dLogits->ld, (int)matR->rows, (int)matR->cols, (int)(matR->nnz / matR->rows),
                          rule->score == B200SP_ROUTE_SIGMOID, rule->renormalise, rule->scale, static_cast<const int *>(matR->indices),
                          matR->values, dValues->values, matR->valueType, dValues->valueType, dLogits->values};
    const cudaError_t e = WithPer(a.experts, [&](auto per) {
        return WithType(logits->valueType, [&](auto in) {
            constexpr int kPer = decltype(per)::value;
            b200sp_note_launches(1);
            return b200sp::LaunchChained(RouteGradKernel<decltype(in), kPer>, RouteBlocks<kPer>(a.tokens), 32 * kRouteWarps<kPer>, 0,
                                         handle->stream, a);
        });
    });
    return Finished(e, "b200spRouteGrad");
}

}  // extern "C"
