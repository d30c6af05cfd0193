// What the token operators on the tensor cores share: barriers, copies by TMA, shared-memory operands, accumulators.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace b200sp_tokens {

constexpr int kBlockBytes = 64 * 128;  // MN-major operands of 16 bits: 64 rows along the sum, 64 elements along the tile

__device__ __forceinline__ uint32_t Shared(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void BarInit(uint64_t *bar, int count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(Shared(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void BarExpect(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(Shared(bar)), "r"(bytes) : "memory");
}
// The barrier in the shared memory of the cluster's first CTA.
__device__ __forceinline__ uint32_t LeadersBar(uint64_t *bar)
{
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(Shared(bar)));
    return at;
}
// Of this CTA or another one of the cluster.  What it orders is read from the arriving CTA's own memories by the tensor cores: tensor memory, or
// shared memory that a proxy fence has handed over.  (A release at cluster scope waits for every access of the SM, 1600 clocks.)
__device__ __forceinline__ void BarArriveAt(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool BarTry(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(Shared(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool BarWait(uint64_t *bar, uint32_t parity, long long limit)
{
    if (BarTry(bar, parity)) return true;
    const long long t0 = clock64();
    while (!BarTry(bar, parity))
        if (clock64() - t0 > limit) return false;
    return true;
}
// One lane of the warp, always the same.  Requests and products are left to it inside code that the whole warp runs, so that their
// operands stay in uniform registers.
__device__ __forceinline__ bool Elected()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// By a whole warp, of which one lane asks: all of its lanes go on, or none.
__device__ __forceinline__ bool BarWaitWarp(uint64_t *bar, uint32_t parity, long long limit)
{
    bool ok = true;
    if ((threadIdx.x & 31) == 0) ok = BarWait(bar, parity, limit);
    return __all_sync(0xffffffffu, ok);
}
// All CTAs of a cluster meet.  Like all `.aligned` instructions it is for whole warps: lanes that have gone different ways come together before it.
__device__ __forceinline__ void ClusterMeet()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Tensor memory that some threads have used and others go on with (or free): the ones order what they did before a barrier, the others what they do after it.
__device__ __forceinline__ void TensorBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void TensorAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// bar: of this CTA, or with a pair of the first.
template <bool kPair> __device__ __forceinline__ void CopyTile3(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar)
{
    if constexpr (kPair)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                         dst),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
}
// 16 bytes of a row, of which the first `bytes` exist and the others arrive as zeros.
__device__ __forceinline__ void CopyPiece(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Shared-memory operands.  K-major: rows of 128 bytes along the sum, eight of them 1024 bytes.  MN-major: rows of 64 elements along the
// tile, eight along the sum 1024 bytes, the next 64 elements a block further.
__device__ __forceinline__ uint64_t OperandAt(uint32_t at, bool alongTile)
{
    const uint64_t leading = alongTile ? kBlockBytes >> 4 : 1, stride = 1024 >> 4;
    return (uint64_t)((at & 0x3ffff) >> 4) | leading << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}
// Arrives, in both CTAs of a pair, when the products so far are complete.
template <bool kPair> __device__ __forceinline__ void MmaCommit(uint64_t *bar)
{
    if constexpr (kPair)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(Shared(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(Shared(bar)) : "memory");
}
__device__ __forceinline__ void LoadColumns32(uint32_t at, float (&v)[32])
{
    uint32_t r[32];
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// The stages in turn, and the parity that a wait for one is for.
struct Ring {
    int stage = 0, round = 0;
    __device__ __forceinline__ void Next(int stages) { On(1, stages); }
    __device__ __forceinline__ void On(int by, int stages)
    {
        for (stage += by; stage >= stages; stage -= stages) ++round;
    }
    __device__ __forceinline__ uint32_t Filled() const { return (uint32_t)round & 1u; }
    __device__ __forceinline__ uint32_t Emptied() const { return (uint32_t)(round - 1) & 1u; }  // not in the first round
};

// ---------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled Encoder()
{
    static const EncodeTiled encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found{};
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(fn) : nullptr;
    }();
    return encode;
}

}  // namespace b200sp_tokens
