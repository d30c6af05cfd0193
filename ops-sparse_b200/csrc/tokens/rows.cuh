// Rows by warps: a warp's lanes lie side by side on a stretch of a row, 256 elements, eight a lane.
#pragma once

#include <type_traits>

#include "tokens/common.cuh"

namespace b200sp_tokens {

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

constexpr int kStretch = 256;

// Eight of a lane's elements of the stretch that starts at column c0, as they lie in memory.  kVector (rows start on 16 bytes): neighbours; else one of
// every 32, so that what the warp asks for at once lies side by side all the same.  Columns past the last are read as zeros, and not stored.
template <typename T> struct __align__(16) Raw {
    static constexpr int kWords = 8 * (int)sizeof(T) / 4;
    uint32_t w[kWords];
    template <bool kVector> __device__ __forceinline__ void Load(const T *row, int c0, int lane, int width)
    {
        const int at = kVector ? c0 + lane * 8 : c0 + lane;
        if (kVector && at + 8 <= width) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = *(reinterpret_cast<const uint4 *>(row + at) + i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
            return;
        }
        constexpr int kStep = kVector ? 1 : 32;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = at + i * kStep < width ? *reinterpret_cast<const uint32_t *>(row + at + i * kStep) : 0u;
            } else {
                const uint32_t low = at + 2 * i * kStep < width ? *reinterpret_cast<const uint16_t *>(row + at + 2 * i * kStep) : 0u;
                const uint32_t high = at + (2 * i + 1) * kStep < width ? *reinterpret_cast<const uint16_t *>(row + at + (2 * i + 1) * kStep) : 0u;
                w[i] = low | high << 16;
            }
        }
    }
    template <bool kVector> __device__ __forceinline__ void Store(T *row, int c0, int lane, int width) const
    {
        const int at = kVector ? c0 + lane * 8 : c0 + lane;
        if (kVector && at + 8 <= width) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i)
                *(reinterpret_cast<uint4 *>(row + at) + i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            return;
        }
        constexpr int kStep = kVector ? 1 : 32;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (at + i * kStep >= width) break;
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t *>(row + at + i * kStep) = w[i];
            else *reinterpret_cast<uint16_t *>(row + at + i * kStep) = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
    __device__ __forceinline__ float At(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return ToFloat(reinterpret_cast<const T *>(w)[i]);
    }
    __device__ __forceinline__ void Floats(float (&v)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = At(i);
    }
    __device__ __forceinline__ void Set(const float (&v)[8])
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
            else w[i] = TwoFromFloats<T>(v[2 * i], v[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void Zero()
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    // The bits of the largest absolute value so far, of two elements of 16 bits side by side; a NaN's are the largest.
    __device__ __forceinline__ uint32_t Top(uint32_t so) const
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) so = sizeof(T) == 4 ? max(so, w[i] & 0x7fffffffu) : __vmaxu2(so, w[i] & 0x7fff7fffu);
        return so;
    }
    // Those of f32.
    __device__ static __forceinline__ uint32_t TopOf(uint32_t so)
    {
        if constexpr (sizeof(T) == 4) return so;
        const uint16_t bits = (uint16_t)max(so & 0xffffu, so >> 16);
        return __float_as_uint(ToFloat(*reinterpret_cast<const T *>(&bits)));
    }
};
// Eight bytes of a stretch.
template <bool kVector> __device__ __forceinline__ void StoreBytes(int8_t *row, int c0, int lane, int width, uint2 words)
{
    const int at = kVector ? c0 + lane * 8 : c0 + lane;
    if (kVector && at + 8 <= width) {
        *reinterpret_cast<uint2 *>(row + at) = words;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (at + (kVector ? i : 32 * i) < width) row[at + (kVector ? i : 32 * i)] = (int8_t)((i < 4 ? words.x : words.y) >> (8 * (i & 3)));
}

// m: the bits of the largest absolute value of a row, whose numbers of 8 bits are whole multiples of Scale().  T: what the row is of.
template <typename T> struct EightBits {
    uint32_t bits;
    float top, up, by;
    bool none, far;  // zeros, or a row that is not finite; one that is taken `up` times as large
    __device__ __forceinline__ explicit EightBits(uint32_t m) : bits(m)
    {
        none = m == 0 || m >= 0x7f800000u;
        // A row of very large or small values is taken as if the largest were near 1, which is exact where it matters: nothing leaves f32's range.
        const int exponent = min(max((int)(m >> 23) - 127, -120), 120);
        far = exponent < -60 || exponent > 60;
        up = far ? __uint_as_float((uint32_t)(127 - exponent) << 23) : 1.0f;
        top = __uint_as_float(m) * up;
        by = __fdividef(1.0f, top);
    }
    __device__ __forceinline__ float Scale() const
    {
        return bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(bits) / 127.0f;
    }
    // Eight values as bytes.  The quotient 127 x / top by one step of Newton's: off by little more than half a step of f32, and exact if it is a half (k + 1/2),
    // as its remainder is then known exactly.  Of 16 bits, 127 x is exact, and a quotient that is no half lies further from one than that
    // (2^s / 4094 at least, where it is some 2^(s + 7)), so that rounding it is rounding the quotient itself.  Of f32 a quotient that comes out as a
    // half may have been near one only: the sign of the remainder says where.  (Halves are not rare: of normal values in bf16 one in 230 is.)
    // It is rounded by 1.5 * 2^23, whose last bits are then the whole number: conversions have a quarter of an addition's rate.
    __device__ __forceinline__ uint2 Of(float (&x)[8]) const
    {
        if (none) return make_uint2(0, 0);
        if (far) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= up;
        }
        constexpr float kRound = 0x1.8p23f;
        int n[8];
        bool half = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = 127.0f * x[i], near = p * by, q = fmaf(Rest(near, p, x[i]), by, near), whole = q + kRound;
            n[i] = __float_as_int(whole);
            if constexpr (sizeof(T) == 4) half |= fabsf(q - (whole - kRound)) == 0.5f;
        }
        if (sizeof(T) == 4 && half) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = 127.0f * x[i], near = p * by, q = fmaf(Rest(near, p, x[i]), by, near), rest = Rest(q, p, x[i]);
                const float whole = __int_as_float(n[i]) - kRound;
                if (fabsf(q - whole) == 0.5f && rest != 0.0f) n[i] = (int)(rest > 0.0f ? ceilf(q) : floorf(q));
            }
        }
        return make_uint2(Four(n[0], n[1], n[2], n[3]), Four(n[4], n[5], n[6], n[7]));
    }
    // 127 x - q top, p = 127 x rounded.
    __device__ __forceinline__ float Rest(float q, float p, float x) const
    {
        const float rest = fmaf(-q, top, p);
        return sizeof(T) == 4 ? rest + fmaf(127.0f, x, -p) : rest;
    }
    __device__ static __forceinline__ uint32_t Four(int a, int b, int c, int d)
    {
        return __byte_perm(__byte_perm((uint32_t)a, (uint32_t)b, 0x0040), __byte_perm((uint32_t)c, (uint32_t)d, 0x0040), 0x5410);
    }
};

}  // namespace b200sp_tokens
