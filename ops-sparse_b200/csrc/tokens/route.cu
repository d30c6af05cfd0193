// b200spRoute, b200spRouteGrad: the k best experts of every token as a CSR matrix, and the gradient of its values.
//
// A warp has a token; its lanes hold the token's logits, 1 to 32 each (expert 32 j + lane).  Every lane sorts its own; then the k experts are
// taken one after the other: the largest key among the lanes' first, the lowest expert that has it, and that lane goes on to its
// next.  Keys are the selection values as unsigned integers of the same order.
// The choice is that of f64 arithmetic.  Without a bias it is made on the logits themselves, which both scores ascend
// with.  With one, p + bias is computed in f32 together with a bound of its error; where another expert lies as near the last
// one taken as the two bounds together, or a group that is kept as near one that is not, the row is done again in
// f64.
// What bounds it are instructions, some 1230 a token: 16,384 tokens, 8 of 256 experts in groups, with a bias 26 us (17.9 MB; 74 % of the issue
// slots), without groups 20, without either 16; the largest of all lanes' experts looked for in every round 52.
#include <cfloat>
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
    int groupSize, groupLanes;  // lanes side by side on a group: a power of two
    unsigned perGroup;          // e / groupSize = e * perGroup >> 20 for e, groupSize <= 1024
    int *offsets, *columns;
    void *values;
};

template <typename Real> struct Limits;
template <> struct Limits<float> {
    static __device__ __forceinline__ float Lowest() { return -INFINITY; }
    static __device__ __forceinline__ float Least() { return -FLT_MAX; }
};
template <> struct Limits<double> {
    static __device__ __forceinline__ double Lowest() { return -(double)INFINITY; }
    static __device__ __forceinline__ double Least() { return -DBL_MAX; }
};

__device__ __forceinline__ float Exp(float v) { return expf(v); }
__device__ __forceinline__ double Exp(double v) { return exp(v); }

__device__ __forceinline__ float Larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double Larger(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float Smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double Smaller(double a, double b) { return fmin(a, b); }

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
__device__ __forceinline__ float ValueOf(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ unsigned long long MaxKey(unsigned long long v)
{
    const uint32_t high = __reduce_max_sync(kAll, (uint32_t)(v >> 32));
    const uint32_t low = __reduce_max_sync(kAll, (uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
    return (unsigned long long)high << 32 | low;
}

// The largest of the warp's, no NaN among them.
__device__ __forceinline__ float LargestOf(float v) { return ValueOf(__reduce_max_sync(kAll, KeyOf(v))); }

__device__ __forceinline__ float Sigmoid(float x)
{
    const float e = expf(-fabsf(x));
    return (x >= 0.0f ? 1.0f : e) / (1.0f + e);
}

// Scores that are divided by their sum may share any factor.  Where the sum is small (by sigmoids, or by exponentials of the difference to
// the row's largest logit) they are taken relative to the largest logit among them: scores below the least f32 still have quotients.
// Above, what is lost is below the least f32 of the quotients, too.
constexpr float kSmall = 0.25f;
__device__ __forceinline__ float FarScore(float x, bool sigmoid, float largest)  // a sigmoid below kSmall: x is negative
{
    return (x == largest ? 1.0f : expf(x - largest)) / (sigmoid ? 1.0f + expf(x) : 1.0f);
}

// Scores of the lanes' logits (masked: -infinity), 0 for the masked.  In f32 a sigmoid is taken from the fast exponential and division: it
// serves the choice alone.  *error: how far they may be from exact ones.
//   sigmoid: __expf is off by 2 + 1.17 |x| units of 2^-23 relative to e^-x, of which p (1 - p) times reaches p: with p (1 - p) <= 1/4 and
//   p (1 - p) |x| < 0.23 less than one unit; the addition and the division bring three more; 8 are allowed.
//   softmax: expf is off by 2 units relative to p, the difference of the logits by |x - most| / 2 (p |x - most| <= 0.4 of the largest score), a
//   sum of kPer + 5 additions by half of that many, the reciprocal and the product by one: at most 24 of the largest score; 32 are
//   allowed.
template <typename Real, int kPer>
__device__ __forceinline__ void Scores(const RouteArgs &a, const float (&x)[kPer], Real (&p)[kPer], float *most, Real *inverse, float *error)
{
    constexpr float kUnit = 1.2e-7f;
    constexpr bool kFast = sizeof(Real) == 4;
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if constexpr (kFast) p[j] = __fdividef(1.0f, 1.0f + __expf(-x[j]));
            else p[j] = 1.0 / (1.0 + exp(-(double)x[j]));
        }
        *error = 8 * kUnit;
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
    *inverse = inv;
    *error = 32 * kUnit * (float)inv;
}

// The selection values: of masked experts, and of those in groups that are not kept, -infinity.  Returns whether f32 can not tell
// which groups are kept.
template <typename Real, int kPer>
__device__ __forceinline__ bool Values(const RouteArgs &a, const float (&x)[kPer], const Real (&p)[kPer], float error, void *sRow, int lane,
                                       Real (&s)[kPer])
{
    const Real nothing = Limits<Real>::Lowest();
    bool unsure = false;
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[j] = (Real)x[j];
    if (a.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = 32 * j + lane;
            const float b = e < a.experts ? __ldg(a.bias + e) : -INFINITY;
            s[j] = x[j] == -INFINITY || !(b > -INFINITY) ? nothing : p[j] + (Real)b;
        }
    }
    if (a.groups == 1) return false;
    // Lanes side by side on a group: the two best of their experts, then of the group.
    Real *const sValues = static_cast<Real *>(sRow);
    const bool sums = a.top2 != 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int e = 32 * j + lane;
        const Real v = sums && a.bias == nullptr ? (x[j] == -INFINITY ? nothing : p[j]) : s[j];
        if (e < a.experts) sValues[e + (e >> 5)] = v;
    }
    __syncwarp();
    const int wide = a.groupLanes, group = lane / wide, size = a.groupSize;
    Real first = nothing, second = nothing;
    if (group < a.groups) {
        for (int i = lane % wide; i < size; i += wide) {
            const int e = group * size + i;
            const Real v = sValues[e + (e >> 5)];
            second = Larger(second, Smaller(first, v));
            first = Larger(first, v);
        }
    }
    for (int d = 1; d < wide; d <<= 1) {
        const Real f = __shfl_xor_sync(kAll, first, d), t = __shfl_xor_sync(kAll, second, d);
        second = Larger(Larger(second, t), Smaller(first, f));
        first = Larger(first, f);
    }
    __syncwarp();  // the values may be written again
    // two of the lowest f32 are no masked group
    const Real value = sums && second > nothing ? Larger(first + second, Limits<Real>::Least()) : first;
    // lane g < groups: group g
    const Real own = __shfl_sync(kAll, value, (lane * wide) & 31), mine = lane < a.groups ? own : nothing;
    int place = 0;
    for (int g = 0; g < a.groups; ++g) {
        const Real o = __shfl_sync(kAll, mine, g);
        place += o > mine || (o == mine && g < lane);
    }
    const bool kept = lane < a.groups && place < a.kept;
    const unsigned open = __ballot_sync(kAll, kept);
    if (sizeof(Real) == 4 && (a.bias != nullptr || sums)) {
        // The last group kept, and the first that is not.  Off are two scores of each, and by half a unit of 2^-23 what rounds: the two values
        // and their sum.  A value with its bias may be far larger than the sum, and any group the one that is off: the largest terms count.
        const uint32_t key = KeyOf((float)mine);
        const float least = ValueOf(__reduce_min_sync(kAll, kept ? key : ~0u));
        const float other = ValueOf(__reduce_max_sync(kAll, lane < a.groups && !kept ? key : KeyOf(-INFINITY)));
        const bool finite = first > nothing && first < (Real)INFINITY;  // infinite ones are exact
        const float terms = finite ? fabsf((float)first) + (sums && second > nothing ? fabsf((float)second) : 0.0f) : 0.0f;
        const float most = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(terms)));
        unsure = other > -INFINITY && !(least - other > 4 * error + 4.8e-7f * most);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int e = 32 * j + lane;
        if (!(open >> (e * a.perGroup >> 20 & 31) & 1)) s[j] = nothing;
    }
    return unsure;
}

// Lane i < k has the i-th expert taken.
struct Chosen {
    int expert;
    bool weightless;  // it has no selection value
};

// By the f64 values, one expert after the other.
template <int kPer> __device__ __noinline__ Chosen ChooseExactly(const RouteArgs &a, const float *sLogits, void *sRow, int lane)
{
    float x[kPer], most, error;
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = sLogits[32 * j + lane];
    double p[kPer], s[kPer], inverse;
    Scores<double, kPer>(a, x, p, &most, &inverse, &error);
    Values<double, kPer>(a, x, p, error, sRow, lane, s);
    Chosen c{-1, false};
    for (int i = 0; i < a.k; ++i) {
        unsigned long long best = 0;
        int at = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const unsigned long long key = 32 * j + lane < a.experts && s[j] == s[j] ? KeyOf(s[j]) : 0;
            if (key > best) {
                best = key;
                at = j;
            }
        }
        const unsigned long long top = MaxKey(best);
        const unsigned e = __reduce_min_sync(kAll, best == top && top != 0 ? 32u * at + lane : ~0u);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (e == 32u * j + lane) s[j] = NAN;  // taken
        if (lane == i) c = {(int)e, top == KeyOf(Limits<double>::Lowest())};
    }
    return c;
}

// Sorts the lane's keys, the largest first, with their places; of equal ones the lower place first: neighbours are exchanged, up to eight
// keys; more by Batcher's odd-even merge sort, which compares the places of equal keys.
template <int kPer> __device__ __forceinline__ void SortDown(uint32_t (&key)[kPer], int (&place)[kPer])
{
    auto exchange = [&](int u, int v, bool swap) {
        const uint32_t high = max(key[u], key[v]), low = min(key[u], key[v]);
        const int pu = swap ? place[v] : place[u], pv = swap ? place[u] : place[v];
        key[u] = high, key[v] = low, place[u] = pu, place[v] = pv;
    };
    if constexpr (kPer <= 8) {
#pragma unroll
        for (int round = 0; round < kPer; ++round)
#pragma unroll
            for (int i = round & 1; i + 1 < kPer; i += 2) exchange(i, i + 1, key[i + 1] > key[i]);
    } else {
#pragma unroll
        for (int p = 1; p < kPer; p *= 2)
#pragma unroll
            for (int k = p; k >= 1; k /= 2)
#pragma unroll
                for (int j = k % p; j + k < kPer; j += 2 * k)
#pragma unroll
                    for (int i = 0; i < k; ++i) {
                        const int u = i + j, v = i + j + k;
                        if (v < kPer && u / (2 * p) == v / (2 * p)) exchange(u, v, key[v] > key[u] || (key[v] == key[u] && place[v] < place[u]));
                    }
    }
}

template <typename In, typename Out, int kPer> __global__ void __launch_bounds__(32 * kRouteWarps<kPer>) RouteKernel(const RouteArgs a)
{
    // of a warp: its selection values by expert, a word apart every 32 (f64 too), and its logits
    __shared__ __align__(8) double sRows[kRouteWarps<kPer>][33 * kPer];
    __shared__ float sAllLogits[kRouteWarps<kPer>][32 * kPer];
    b200sp::WaitForPrevious();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long token = (long long)blockIdx.x * kRouteWarps<kPer> + warp;
    if (token >= a.tokens) return;
    uint2 *const sList = reinterpret_cast<uint2 *>(sRows[warp]) + lane;  // the lane's sorted keys and experts, 32 apart
    const In *const row = static_cast<const In *>(a.logits) + token * a.ld;
    float *const sLogits = sAllLogits[warp];
    float x[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        x[j] = 32 * j + lane < a.experts ? ToFloat(row[32 * j + lane]) : -INFINITY;
        x[j] = fmaxf(x[j], -INFINITY);  // NaN is masked, too
        sLogits[32 * j + lane] = x[j];
    }
    __syncwarp();
    float p[kPer], s[kPer], most = 0.0f, inverse = 0.0f, error = 0.0f;
    const bool scored = !a.sigmoid || a.bias != nullptr || (a.groups > 1 && a.top2);  // without, the choice goes by the logits alone
    if (scored) Scores<float, kPer>(a, x, p, &most, &inverse, &error);
    bool unsure = Values<float, kPer>(a, x, p, error, sRows[warp], lane, s);
    uint32_t key[kPer];
    int place[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        key[j] = 32 * j + lane < a.experts ? KeyOf(s[j]) : 0;
        place[j] = j;
    }
    SortDown<kPer>(key, place);
    // The lists lie in shared memory; a lane has its first in hand.
#pragma unroll
    for (int j = 1; j < kPer; ++j) sList[32 * (j - 1)] = make_uint2(key[j], 32u * place[j] + lane);
    sList[32 * (kPer - 1)] = make_uint2(0u, 0u);
    uint2 head = make_uint2(key[0], 32u * place[0] + lane);
    int at = 0;
    const uint32_t nothing = KeyOf(-INFINITY);
    Chosen c{-1, false};
    uint32_t top = 0, taken = 0;  // of the last one, of the lane's
    unsigned e = 0;
    for (int i = 0; i < a.k; ++i) {
        top = __reduce_max_sync(kAll, head.x);
        e = __reduce_min_sync(kAll, head.x == top ? head.y : ~0u);
        if (lane == i) c = {(int)e, top == nothing}, taken = top;
        if (head.y == e && head.x != 0) head = sList[at], at += 32;
    }
    if (a.bias != nullptr) {
        // Experts left out as near the last one taken as f32 tells: the choice is certain only where they, and those taken that are as near,
        // all have its logit and bias.  (Equals of the last that are left out may be above another one taken.)
        const float last = ValueOf(top), room = 2 * error + 4.8e-7f * fabsf(last);
        const uint32_t near = top == nothing ? ~0u : KeyOf(last - room);
        const auto differs = [&](unsigned other) { return !(sLogits[other] == sLogits[e] && __ldg(a.bias + other) == __ldg(a.bias + e)); };
        if (__any_sync(kAll, head.x > nothing && head.x >= near)) {
            unsure |= lane < a.k && taken <= KeyOf(last + room) && differs(c.expert);
            do {
                if (head.x > nothing && head.x >= near) {
                    unsure |= differs(head.y);
                    head = sList[at], at += 32;
                }
            } while (__any_sync(kAll, head.x > nothing && head.x >= near));
        }
    }
    if (__any_sync(kAll, unsure)) c = ChooseExactly<kPer>(a, sLogits, sRows[warp], lane);
    // the weights, of the experts taken alone; their places by column
    const bool weighs = c.expert >= 0 && !c.weightless;
    const float own = weighs ? sLogits[c.expert] : -INFINITY;
    float w = 0.0f;
    if (weighs) w = a.sigmoid ? Sigmoid(own) : own == most ? 1.0f : expf(own - most);
    float by = a.scale;
    if (a.renormalise) {
        float sum = WarpSum(w);
        if (sum < kSmall) {
            const float largest = LargestOf(own);
            if (weighs) w = FarScore(own, a.sigmoid, largest);
            sum = WarpSum(w);
        }
        by = sum > 0 ? a.scale / sum : 0.0f;
    } else if (!a.sigmoid) {
        w *= inverse;
    }
    int to = 0;
    for (int i = 0; i < a.k; ++i) to += __shfl_sync(kAll, c.expert, i) < c.expert;
    if (lane < a.k) {
        a.columns[token * a.k + to] = c.expert;
        static_cast<Out *>(a.values)[token * a.k + to] = FromFloat<Out>(w * by);
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

// A warp has a token.  What bounds it is the latency of its chain: columns, their logits, sums over the lanes, the row through shared memory.
// 16,384 tokens, 8 of 128 experts, bf16: 5.5 us renormalised softmax, 7.2 sigmoid, 9.0 with all logits (softmax as it is).
// Lane i has entry i of the token's row.  With q the weights over scale and g their gradients, scale times
//   softmax, renormalised   dx = q (g - sum g q): the softmax of the chosen logits alone
//   sigmoid, renormalised   dx = q (g - sum g q) (1 - s)
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
            g = LoadAs(a.grad, i, a.gradType);
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
        for (int j = 0; j < kPer; ++j) sRow[32 * j + lane] = -a.scale * v[j] * inv * dot;
        dx = p * (g - dot);
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) sRow[32 * j + lane] = 0.0f;
        if (a.sigmoid) {
            float s = col < 0 ? 0.0f : Sigmoid(x);
            const float rest = col < 0 ? 0.0f : 1.0f / (1.0f + expf(x));  // 1 - the score, exactly enough where that is near 1
            if (a.renormalise) {
                float sum = WarpSum(s), dot = WarpSum(g * s);
                if (sum < kSmall) {
                    const float largest = LargestOf(x);
                    if (col >= 0) s = FarScore(x, true, largest);
                    sum = WarpSum(s), dot = WarpSum(g * s);
                }
                dx = sum > 0 ? (g - dot / sum) / sum * s * rest : 0.0f;
            } else {
                dx = g * s * rest;
            }
        } else {
            const float m = WarpMax(x);
            const float e = col < 0 ? 0.0f : x == m ? 1.0f : expf(x - m);
            const float sum = WarpSum(e), q = sum > 0 ? e / sum : 0.0f;
            dx = q * (g - WarpSum(g * q));
        }
    }
    __syncwarp();
    if (col >= 0) sRow[col] = a.scale * dx;
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
    if (!OnBoundary(R->offsets, 4) || !OnBoundary(R->indices, 4) || !OnBoundary(R->values, BytesOf(R->valueType))) return ACL_SPARSE_STATUS_INVALID_VALUE;
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
        if (bias->magic != b200sp::kDnVecMagic || bias->size != matR->cols || !OnBoundary(bias->values, 4)) return ACL_SPARSE_STATUS_INVALID_VALUE;
        if (bias->valueType != ACL_FLOAT) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    const OnDevice device(handle);
    RouteArgs a{logits->values, bias != nullptr ? static_cast<const float *>(bias->values) : nullptr, logits->ld, (int)matR->rows,
                (int)matR->cols, (int)(matR->nnz / matR->rows), rule->score == B200SP_ROUTE_SIGMOID, rule->groups, rule->groupsKept,
                rule->groupScore == B200SP_GROUP_TOP2, rule->renormalise, rule->scale, 0, 0, 0, static_cast<int *>(matR->offsets),
                static_cast<int *>(matR->indices), matR->values};
    {
        // R's columns are written: no buffer holds their order any more.  (A captured call has not written them yet.)
        std::lock_guard<std::mutex> lock(matR->expertsMutex);
        if (Captures(handle->stream)) matR->experts.stale = true;
        else matR->experts = {};
    }
    if (a.kept == a.groups) a.groups = a.kept = 1;  // all are kept
    a.groupSize = a.experts / a.groups;
    a.perGroup = ((1u << 20) + a.groupSize - 1) / a.groupSize;
    for (a.groupLanes = 32; a.groupLanes * a.groups > 32;) a.groupLanes /= 2;
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
    if (!OnBoundary(dValues->values, BytesOf(dValues->valueType))) return ACL_SPARSE_STATUS_INVALID_VALUE;
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
