// Rows by warps: a warp's lanes lie side by side on a stretch of a row, kN elements a lane.
#pragma once

#include "tokens/common.cuh"

namespace b200sp_tokens {

// The lane's elements of the stretch that starts at column c0: kVector (rows start on 16 bytes): kN neighbours; else one of every 32, so that
// what the warp asks for at once lies side by side all the same.  Columns past the last are zeros, and not stored.
template <typename T, int kN, bool kVector>
__device__ __forceinline__ void LoadStretch(const T *row, int c0, int lane, int width, float (&v)[kN])
{
    if constexpr (kVector) {
        const int at = c0 + lane * kN;
        if (at + kN <= width) {
            LoadFloats<T, kN, true>(row + at, v);
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = at + i < width ? ToFloat(row[at + i]) : 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = c0 + 32 * i + lane < width ? ToFloat(row[c0 + 32 * i + lane]) : 0.0f;
    }
}
template <typename T, int kN, bool kVector>
__device__ __forceinline__ void StoreStretch(T *row, int c0, int lane, int width, const float (&v)[kN])
{
    if constexpr (kVector) {
        const int at = c0 + lane * kN;
        if (at + kN <= width) {
            StoreFloats<T, kN, true>(row + at, v);
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (at + i < width) row[at + i] = FromFloat<T>(v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (c0 + 32 * i + lane < width) row[c0 + 32 * i + lane] = FromFloat<T>(v[i]);
    }
}

// A value of a type that is known at run time only.
__device__ __forceinline__ float ValueAt(const void *values, aclDataType type, int i)
{
    if (type == ACL_FLOAT16) return __half2float(static_cast<const __half *>(values)[i]);
    if (type == ACL_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(values)[i]);
    return static_cast<const float *>(values)[i];
}
__device__ __forceinline__ void SetValue(void *values, aclDataType type, int i, float v)
{
    if (type == ACL_FLOAT16) static_cast<__half *>(values)[i] = __float2half_rn(v);
    else if (type == ACL_BF16) static_cast<__nv_bfloat16 *>(values)[i] = __float2bfloat16_rn(v);
    else static_cast<float *>(values)[i] = v;
}

// Rows and stretches in turn: `step` units further, without a division.
struct Units {
    long long row;
    int stretch, stretches;
    long long rowStep;
    int stretchStep;
    __device__ __forceinline__ Units(long long first, long long step, int perRow)
        : row(first / perRow), stretch((int)(first % perRow)), stretches(perRow), rowStep(step / perRow), stretchStep((int)(step % perRow))
    {
    }
    __device__ __forceinline__ void Next()
    {
        row += rowStep;
        stretch += stretchStep;
        if (stretch >= stretches) {
            stretch -= stretches;
            ++row;
        }
    }
};

// m: the bits of the largest absolute value of a row.  Numbers of 8 bits are whole multiples of `scale` from there on.
struct EightBits {
    float scale, top, up, by;
    bool none;  // zeros, or a row that is not finite
    __device__ __forceinline__ explicit EightBits(uint32_t m)
    {
        top = __uint_as_float(m);
        none = m == 0 || m >= 0x7f800000u;
        scale = m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : top / 127.0f;
        // 127 / top is no f32 below 2^-121: small rows are taken 2^100 times as large, which is exact
        up = top < 0x1p-100f ? 0x1p100f : 1.0f;
        top *= up;
        by = 127.0f / top;
    }
    // t is off by two roundings, 127 * 2^-23 at most.  Where that could decide, the quotient is taken in f64: 127 x has 31 bits and the divisor 24, so
    // that a quotient which is no half lies further from one than f64 rounds, and a half comes out as it is.
    __device__ __forceinline__ int Of(float x) const
    {
        if (none) return 0;
        const float t = x * up * by, n = rintf(t);
        if (fabsf(t - n) > 0.5f - 0x1p-15f) return (int)rint(127.0 * (double)(x * up) / (double)top);
        return (int)n;
    }
};

}  // namespace b200sp_tokens
