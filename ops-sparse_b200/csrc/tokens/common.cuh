// What the token operators (include/b200sp_tokens.h) share: element types, scalars, argument checks, the handle's device.
#pragma once

#include <atomic>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "b200sp_kernels.h"
#include "common/chained.cuh"
#include "common/internal.h"

namespace b200sp_tokens {

// Positions, columns: what a loop counts to, so that a step further is still an int.
constexpr long long kMostCounted = (1ll << 31) - (1 << 20);

inline size_t AlignUp(size_t v, size_t a) { return (v + a - 1) / a * a; }
inline bool OnBoundary(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool Aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two neighbours in a word.
template <typename T> __device__ __forceinline__ uint32_t TwoFromFloats(float a, float b);
template <> __device__ __forceinline__ uint32_t TwoFromFloats<__half>(float a, float b)
{
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t TwoFromFloats<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// alpha and beta of a call: values, or device pointers to them.
struct Scalars {
    float alpha, beta;
    const float *alphaAt, *betaAt;
    __device__ __forceinline__ float Alpha() const { return alphaAt != nullptr ? __ldg(alphaAt) : alpha; }
    __device__ __forceinline__ float Beta() const { return betaAt != nullptr ? __ldg(betaAt) : beta; }
};
inline Scalars ScalarsOf(const aclsparseContext *handle, const void *alpha, const void *beta)
{
    Scalars s{1.0f, 0.0f, nullptr, nullptr};
    if (handle->pointerMode == ACL_SPARSE_POINTER_MODE_DEVICE) {
        s.alphaAt = static_cast<const float *>(alpha);
        s.betaAt = static_cast<const float *>(beta);
    } else {
        if (alpha != nullptr) s.alpha = *static_cast<const float *>(alpha);
        if (beta != nullptr) s.beta = *static_cast<const float *>(beta);
    }
    return s;
}

// kN neighbouring elements as floats; kVector: they start on a multiple of 16 bytes (and fill 16 or 32).
template <typename T, int kN, bool kVector> __device__ __forceinline__ void LoadFloats(const T *at, float (&v)[kN])
{
    if constexpr (kVector) {
        static_assert(kN * sizeof(T) % 16 == 0);
        uint4 raw[kN * sizeof(T) / 16];
#pragma unroll
        for (int i = 0; i < (int)(kN * sizeof(T) / 16); ++i) raw[i] = *(reinterpret_cast<const uint4 *>(at) + i);
        const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = ToFloat(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = ToFloat(at[i]);
    }
}
template <typename T, int kN, bool kVector> __device__ __forceinline__ void StoreFloats(T *at, const float (&v)[kN])
{
    if constexpr (kVector) {
        static_assert(kN * sizeof(T) % 16 == 0);
        uint32_t words[kN * sizeof(T) / 4];
#pragma unroll
        for (int i = 0; i < (int)(kN * sizeof(T) / 4); ++i) {
            if constexpr (sizeof(T) == 4) words[i] = __float_as_uint(v[i]);
            else words[i] = TwoFromFloats<T>(v[2 * i], v[2 * i + 1]);
        }
#pragma unroll
        for (int i = 0; i < (int)(kN * sizeof(T) / 16); ++i)
            *(reinterpret_cast<uint4 *>(at) + i) = make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) at[i] = FromFloat<T>(v[i]);
    }
}

inline bool IsFloatType(aclDataType t) { return t == ACL_FLOAT || t == ACL_FLOAT16 || t == ACL_BF16; }
inline int BytesOf(aclDataType t) { return t == ACL_FLOAT ? 4 : 2; }

// Rows of a descriptor start on multiples of 16 bytes.
inline bool RowsAligned(const aclsparseDnMatDescr *m)
{
    return Aligned16(m->values) && m->ld * BytesOf(m->valueType) % 16 == 0;
}

// What every dense operand has to be.  (A descriptor has at least one row and one column.)
inline aclsparseStatus_t CheckDense(const aclsparseDnMatDescr *m)
{
    if (m == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (m->order != ACL_SPARSE_ORDER_ROW || !IsFloatType(m->valueType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (m->rows > INT32_MAX || m->cols > kMostCounted || m->ld > INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (m->values == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (!OnBoundary(m->values, BytesOf(m->valueType))) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

// Calls f with a value of the element type.
template <typename F> auto WithType(aclDataType t, F &&f)
{
    switch (t) {
        case ACL_FLOAT16: return f(__half{});
        case ACL_BF16: return f(__nv_bfloat16{});
        default: return f(float{});
    }
}

// The handle's device is the current one while this lives.
class OnDevice {
public:
    explicit OnDevice(const aclsparseContext *handle)
    {
        if (cudaGetDevice(&before_) != cudaSuccess || before_ == handle->device) return;
        changed_ = cudaSetDevice(handle->device) == cudaSuccess;
    }
    ~OnDevice()
    {
        if (changed_) (void)cudaSetDevice(before_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

private:
    int before_ = 0;
    bool changed_ = false;
};

// A buffer that a call is about to write: analyses that lie in it are stale.  0 without memory for the note.
inline uint64_t NoteWrite(const void *buffer) noexcept
{
    try {
        return b200sp::NoteBufferWrite(buffer);
    } catch (...) {
        return 0;
    }
}

// Lets a kernel use `bytes` of shared memory on the current device, where no call has done so yet.
template <auto kKernel> cudaError_t AllowShared(int bytes)
{
    static std::atomic<bool> done[64] = {};
    int device = 0;
    const cudaError_t got = cudaGetDevice(&device);
    if (got != cudaSuccess || device < 0 || device >= 64) return cudaErrorInvalidDevice;
    if (done[device].load(std::memory_order_relaxed)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done[device].store(true, std::memory_order_relaxed);
    return e;
}

// Whether calls on the stream are recorded and not run.
inline bool Captures(cudaStream_t stream)
{
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &capture) == cudaSuccess) return capture != cudaStreamCaptureStatusNone;
    (void)cudaGetLastError();
    return false;
}

inline aclsparseStatus_t Finished(cudaError_t e, const char *call)
{
    if (e == cudaSuccess) return ACL_SPARSE_STATUS_SUCCESS;
    B200SP_LOGE("%s: launch failed (%s)", call, cudaGetErrorString(e));
    (void)cudaGetLastError();
    return ACL_SPARSE_STATUS_EXECUTION_FAILED;
}

}  // namespace b200sp_tokens
