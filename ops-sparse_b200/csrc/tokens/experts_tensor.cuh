// The experts' products on the tensor cores: included by experts.cu.
//
// A tile is 128 columns of Y (of an expert's matrix, the rows "M" of tcgen05.mma) by up to 256 entries of the expert (its "N"),
// that is Y^T = op(W) X^T: with few entries, as when single tokens are served, N shrinks to 16 and what moves is W,
// at full width; the accumulator's lanes are then columns of Y, and a store is 32 of them for one entry.
// The gradient's tile is 128 rows of dW by up to 256 of its columns, summed over the expert's entries.
//
// One CTA per SM walks over the tiles of all experts.  One warp requests: W by tiles, rows of X (and dY) by
// tile::gather4, four rows of 128 bytes that may lie anywhere, so that nothing is laid out in between; a row
// past the tile's last is asked for past the matrix's end and arrives as zeros.  One thread starts the products, four warps
// empty the accumulators, of which there are two: the next tile is summed meanwhile.
// Operands arrive in rows of 128 bytes, swizzled: K-major where those run along the sum (X; W with opW = T), MN-major
// where they run along the tile (W with opW = N; both of the gradient's).
//
// Every wait is bounded.  One that ran out ends its warp's work, raises the flag of b200spExpertsError and leaves rows of the
// output unwritten; nothing waits for ever, and tensor memory is freed when copies and products in flight have had time to
// land.
#pragma once

#include <cuda.h>

constexpr int kMmaRows = 128;                      // of a tile: lanes of tensor memory
constexpr int kMmaDepth = 64;                      // of a stage: 128 bytes
constexpr int kMmaColsMost = 256;                  // of a tile: an accumulator's columns
constexpr int kMmaABytes = kMmaRows * kMmaDepth * 2;
constexpr int kMmaBlockBytes = kMmaDepth * 128;    // MN-major: 64 rows along the sum, 64 elements along the tile
constexpr int kMmaShared = 208 << 10;              // for stages
constexpr int kMmaStagesMost = 12;
constexpr int kMmaThreads = 192;                   // warp 0 requests, 1 multiplies, 2 ... 5 store
constexpr long long kMmaWaitCycles = 4'000'000'000;  // two seconds

enum class Mode { kProductT, kProductN, kGrad };

struct MmaArgs {
    const int *offsets, *entries, *rows;
    void *out;
    long long ldo;
    int experts, n, d;
    int byEntry;
    int rowsA, rowsB;      // rows of what is gathered: dY, X.  One more is past the end
    int colsMost;          // of a tile
    int stages, stageBytes;
    Scalars sc;
    long long waitCycles;
    unsigned extraTx;      // bytes expected on every barrier beyond those copied (0 outside the wait test)
};

__device__ int gExpertsError = 0;

__device__ __forceinline__ uint32_t Shared(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void BarInit(uint64_t *bar, int count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(Shared(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void BarExpect(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(Shared(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void BarArrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(Shared(bar)) : "memory");
}
__device__ __forceinline__ bool BarTry(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
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
// By a whole warp: all of its lanes go on, or none.
__device__ __forceinline__ bool BarWaitWarp(uint64_t *bar, uint32_t parity, long long limit)
{
    return __all_sync(0xffffffffu, BarWait(bar, parity, limit));
}
__device__ __forceinline__ void CopyTile3(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(Shared(bar))
                 : "memory");
}
__device__ __forceinline__ void CopyRows4(uint32_t dst, const CUtensorMap *map, int x, const int (&row)[4], uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
                     dst),
                 "l"(map), "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(Shared(bar))
                 : "memory");
}
// Shared-memory operands.  K-major: rows of 128 bytes along the sum, eight of them 1024 bytes.  MN-major: rows of 64 elements along the
// tile, eight along the sum 1024 bytes, the next 64 elements a block further.
__device__ __forceinline__ uint64_t OperandAt(uint32_t at, bool alongTile)
{
    const uint64_t leading = alongTile ? kMmaBlockBytes >> 4 : 1, stride = 1024 >> 4;
    return (uint64_t)((at & 0x3ffff) >> 4) | leading << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void Mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void MmaCommit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(Shared(bar)) : "memory");
}
__device__ __forceinline__ void LoadColumns16(uint32_t at, float (&v)[16])
{
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// What a tile is: columns [f0, f0 + 128) of Y for entries [first, first + many) of the expert, or rows [f0, ...) and columns
// [first, first + many) of its gradient.
struct MmaTile {
    int expert, f0, first, many, steps;
};

template <Mode kMode> struct Tiles {
    const MmaArgs &a;
    const int *sStart;  // [experts + 2]: the first tile of every expert, and of the group of no expert
    int fTiles;

    __device__ __forceinline__ int Groups() const { return kMode == Mode::kGrad ? a.experts : a.experts + 1; }
    __device__ __forceinline__ int Features() const { return kMode == Mode::kProductN ? a.d : a.n; }
    // Tiles of `count` entries side by side, nearly equal.
    __device__ __forceinline__ int Across(int count) const { return (count + a.colsMost - 1) / a.colsMost; }
    __device__ __forceinline__ int Count(int lo, int hi) const
    {
        return fTiles * (kMode == Mode::kGrad ? (a.d + a.colsMost - 1) / a.colsMost : Across(hi - lo));
    }
    __device__ __forceinline__ MmaTile At(int t) const
    {
        int lo = 0, hi = Groups();
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sStart[mid] <= t) lo = mid;
            else hi = mid;
        }
        MmaTile m;
        m.expert = lo;
        const int within = t - sStart[lo], from = __ldg(a.offsets + lo), count = __ldg(a.offsets + lo + 1) - from;
        const int length = kMode == Mode::kGrad ? a.d : count;
        const int across = (length + a.colsMost - 1) / a.colsMost;
        // kGrad: whole blocks of 64 columns; products: sixteens of entries
        const int unit = kMode == Mode::kGrad ? 64 : 16;
        const int per = ((length + across - 1) / across + unit - 1) / unit * unit;
        const int c = within % across * per;
        m.f0 = within / across * kMmaRows;
        m.first = kMode == Mode::kGrad ? c : from + c;
        m.many = min(per, length - c);
        if (kMode == Mode::kGrad) m.steps = (count + kMmaDepth - 1) / kMmaDepth;
        else m.steps = lo < a.experts && m.many > 0 ? ((kMode == Mode::kProductT ? a.d : a.n) + kMmaDepth - 1) / kMmaDepth : 0;
        return m;
    }
};

template <typename T, typename Out, Mode kMode>
__global__ void __launch_bounds__(kMmaThreads, 1) ExpertsTensorKernel(const MmaArgs a, const __grid_constant__ CUtensorMap mapA,
                                                                      const __grid_constant__ CUtensorMap mapB)
{
    extern __shared__ unsigned char sRaw[];
    __shared__ uint64_t sFull[kMmaStagesMost], sEmpty[kMmaStagesMost], sDone[2], sFree[2], sLast;
    __shared__ uint32_t sTmem;
    __shared__ int sStart[kMaxExperts + 2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = (Shared(sRaw) + 1023u) & ~1023u;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Shared(&sTmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int s = 0; s < a.stages; ++s) {
            BarInit(sFull + s, 1);
            BarInit(sEmpty + s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            BarInit(sDone + i, 1);
            BarInit(sFree + i, 4);
        }
        BarInit(&sLast, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    b200sp::WaitForPrevious();
    const Tiles<kMode> tiles{a, sStart, ((kMode == Mode::kProductN ? a.d : a.n) + kMmaRows - 1) / kMmaRows};
    const int groups = tiles.Groups();
    for (int e = tid; e < groups; e += kMmaThreads) sStart[e] = tiles.Count(__ldg(a.offsets + e), __ldg(a.offsets + e + 1));
    __syncthreads();
    if (warp == 0) {
        int run = 0;
        for (int e0 = 0; e0 <= groups; e0 += 32) {
            const int own = e0 + lane < groups ? sStart[e0 + lane] : 0;
            int incl = own;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += up;
            }
            if (e0 + lane <= groups) sStart[e0 + lane] = run + incl - own;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sTmem;
    const int all = sStart[groups];
    bool failed = false;

    if (warp == 0) {
        int asked = 0;  // stages
        // a stage that is free, or false
        auto stage = [&](uint32_t bytes) {
            const int s = asked % a.stages, use = asked / a.stages;
            if (use > 0 && !BarWaitWarp(sEmpty + s, (uint32_t)(use - 1) & 1u, a.waitCycles)) return false;
            if (lane == 0) BarExpect(sFull + s, bytes + a.extraTx);
            __syncwarp();
            ++asked;
            return true;
        };
        for (int t = blockIdx.x; t < all && !failed; t += gridDim.x) {
            const MmaTile m = tiles.At(t);
            if constexpr (kMode != Mode::kGrad) {
                const int gathers = (m.many + 15) / 16 * 4;
                int row[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = 4 * (lane + 32 * h) + i;
                        row[h][i] = at < m.many ? __ldg((a.byEntry ? a.entries : a.rows) + m.first + at) : a.rowsB;
                    }
                for (int k = 0; k < m.steps; ++k) {
                    const int s = asked % a.stages;
                    if (!stage(kMmaABytes + gathers * 512)) {
                        failed = true;
                        break;
                    }
                    const uint32_t at = base + s * a.stageBytes;
                    if (kMode == Mode::kProductT) {
                        if (lane == 0) CopyTile3(at, &mapA, k * kMmaDepth, m.f0, m.expert, sFull + s);
                    } else if (lane < 2) {
                        CopyTile3(at + lane * kMmaBlockBytes, &mapA, m.f0 + 64 * lane, k * kMmaDepth, m.expert, sFull + s);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (lane + 32 * h < gathers)
                            CopyRows4(at + kMmaABytes + (lane + 32 * h) * 512, &mapB, k * kMmaDepth, row[h], sFull + s);
                }
            } else {
                const int from = __ldg(a.offsets + m.expert), to = __ldg(a.offsets + m.expert + 1);
                const int blocks = (m.many + 63) / 64, mine = lane % 16, half = lane / 16;
                int rowA[4], rowB[4];
                auto rows = [&](int k) {  // of the lane's four entries of a step
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = from + k * kMmaDepth + 4 * mine + i;
                        rowA[i] = at < to ? __ldg(a.entries + at) : a.rowsA;
                        rowB[i] = at < to ? (a.byEntry ? rowA[i] : __ldg(a.rows + at)) : a.rowsB;
                    }
                };
                if (m.steps > 0) rows(0);
                for (int k = 0; k < m.steps; ++k) {
                    const int s = asked % a.stages;
                    if (!stage(kMmaABytes + blocks * kMmaBlockBytes)) {
                        failed = true;
                        break;
                    }
                    const uint32_t at = base + s * a.stageBytes + mine * 512;
                    CopyRows4(at + half * kMmaBlockBytes, &mapA, m.f0 + 64 * half, rowA, sFull + s);
                    for (int b = half; b < blocks; b += 2)
                        CopyRows4(at + kMmaABytes + b * kMmaBlockBytes, &mapB, m.first + 64 * b, rowB, sFull + s);
                    if (k + 1 < m.steps) rows(k + 1);
                }
            }
        }
        // copies on their way after a failure: a bounded chance to land
        if (failed && lane == 0)
            for (int i = asked > a.stages ? asked - a.stages : 0; i < asked; ++i)
                (void)BarWait(sFull + i % a.stages, (uint32_t)(i / a.stages) & 1u, a.waitCycles);
    } else if (tid == 32) {
        constexpr bool kAcrossA = kMode != Mode::kProductT, kAcrossB = kMode == Mode::kGrad;
        const uint32_t type = sizeof(T) == 2 && std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
        const uint32_t instr = 1u << 4 | type << 7 | type << 10 | (uint32_t)kAcrossA << 15 | (uint32_t)kAcrossB << 16 | (uint32_t)(kMmaRows >> 4) << 24;
        int used = 0, tile = 0;
        for (int t = blockIdx.x; t < all && !failed; t += gridDim.x) {
            const MmaTile m = tiles.At(t);
            if (m.steps == 0) continue;
            const int acc = tile & 1, turn = tile >> 1;
            if (turn > 0 && !BarWait(sFree + acc, (uint32_t)(turn - 1) & 1u, a.waitCycles)) {
                failed = true;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t shape = instr | (uint32_t)((m.many + 15) / 16 * 16 >> 3) << 17, to = tmem + acc * kMmaColsMost;
            for (int k = 0; k < m.steps; ++k, ++used) {
                const int s = used % a.stages;
                if (!BarWait(sFull + s, (uint32_t)(used / a.stages) & 1u, a.waitCycles)) {
                    failed = true;
                    break;
                }
                const uint32_t at = base + s * a.stageBytes;
#pragma unroll
                for (int i = 0; i < kMmaDepth / 16; ++i)
                    Mma(to, OperandAt(at + i * (kAcrossA ? 2048 : 32), kAcrossA), OperandAt(at + kMmaABytes + i * (kAcrossB ? 2048 : 32), kAcrossB),
                        shape, k > 0 || i > 0);
                MmaCommit(sEmpty + s);
            }
            if (!failed) MmaCommit(sDone + acc);
            ++tile;
        }
        MmaCommit(&sLast);  // when every product started here is complete, also after a failure
        (void)BarWait(&sLast, 0, a.waitCycles);
    } else if (warp >= 2) {
        const int quarter = warp & 3;  // the lanes of tensor memory that the warp may read
        const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
        const int features = kMode == Mode::kProductN ? a.d : a.n;
        int tile = 0;
        for (int t = blockIdx.x; t < all; t += gridDim.x) {
            const MmaTile m = tiles.At(t);
            const int acc = tile & 1, turn = tile >> 1;
            if (m.steps > 0) {
                if (!BarWaitWarp(sDone + acc, (uint32_t)turn & 1u, a.waitCycles)) {
                    failed = true;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                ++tile;
            }
            const int f = m.f0 + quarter * 32 + lane;
            const uint32_t from = tmem + ((uint32_t)quarter << 21) + acc * kMmaColsMost;
            for (int c0 = 0; c0 < m.many; c0 += 16) {
                float v[16] = {};
                if (m.steps > 0) LoadColumns16(from + c0, v);
                if (m.steps > 0 && c0 + 16 >= m.many) {  // all that this warp reads of the accumulator
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) BarArrive(sFree + acc);
                }
                if constexpr (kMode != Mode::kGrad) {
                    const int entry = c0 + (lane & 15) < m.many ? __ldg(a.entries + m.first + c0 + (lane & 15)) : 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const long long row = __shfl_sync(0xffffffffu, entry, i);
                        if (c0 + i >= m.many || f >= features) continue;
                        Out *const to = static_cast<Out *>(a.out) + row * a.ldo + f;
                        float u = alpha * v[i];
                        if (m.steps == 0) u = 0.0f;
                        if (beta != 0.0f) u = fmaf(beta, ToFloat(*to), u);
                        *to = FromFloat<Out>(u);
                    }
                } else if (f < features) {
                    Out *const to = static_cast<Out *>(a.out) + ((long long)m.expert * a.n + f) * a.ldo + m.first + c0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (c0 + i >= m.many) continue;
                        float u = m.steps == 0 ? 0.0f : alpha * v[i];
                        if (beta != 0.0f) u = fmaf(beta, ToFloat(to[i]), u);
                        to[i] = FromFloat<Out>(u);
                    }
                }
            }
        }
    }
    __syncwarp();
    if (failed) atomicExch(&gExpertsError, 1);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

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

// Rows of 64 elements of a matrix, swizzled: four anywhere (gather), or `high` neighbours of one of `deep` stacked matrices.
inline bool MapOf(CUtensorMap *map, aclDataType type, const void *at, long long cols, long long rows, long long ld, int deep, int high)
{
    const EncodeTiled encode = Encoder();
    if (encode == nullptr) return false;
    const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)deep};
    const cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(ld * 2 * rows)};
    const cuuint32_t box[3] = {64, (cuuint32_t)high, 1}, step[3] = {1, 1, 1};
    return encode(map, type == ACL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, deep > 0 ? 3 : 2,
                  const_cast<void *>(at), size, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Entries of a tile: as many as an expert has on average, half as much again for the uneven ones, so that the weights of most experts are
// read by one tile a column block, and stages are no larger than that wants.
inline int TileColumns(long long nnz, long long experts)
{
    const long long want = (nnz * 3 + 2 * experts - 1) / (2 * experts);
    int cols = 32;
    while (cols < kMmaColsMost && cols < want) cols *= 2;
    return cols;
}

long long gExpertsWaitCycles = kMmaWaitCycles;
unsigned gExpertsExtraTx = 0;

template <typename T, typename Out, Mode kMode>
cudaError_t LaunchTensor(MmaArgs a, const CUtensorMap &mapA, const CUtensorMap &mapB, cudaStream_t stream)
{
    a.stageBytes = kMmaABytes + a.colsMost * 128;
    a.stages = std::min(kMmaShared / a.stageBytes, kMmaStagesMost);
    a.waitCycles = gExpertsWaitCycles;
    a.extraTx = gExpertsExtraTx;
    const auto kernel = ExpertsTensorKernel<T, Out, kMode>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMmaShared + 1024);
    if (e != cudaSuccess) return e;
    b200sp_note_launches(1);
    return b200sp::LaunchChained(kernel, (unsigned)b200sp_sm_count(), kMmaThreads, (size_t)(a.stages * a.stageBytes + 1024), stream, a, mapA, mapB);
}
