// Products in 8-bit integers on the tensor cores: included by scaled.cu.
//
// Y^T = W X^T: a tile is 128 channels (rows of W, the rows "M" of tcgen05.mma, kind::i8) by up to 256 rows of X (its "N"), so that with few rows, as
// when single tokens are served, N shrinks and what moves is W.  With experts, whose rows lie side by side, a tile is one expert's.
// One warp requests both operands by TMA, in rows of 128 bytes, swizzled; one starts the products; eight empty the accumulators, of which there are
// two: the next tile is summed meanwhile.  Sums are whole numbers of 32 bits; they are scaled in f32 and rounded once.
//
// Every wait is bounded.  One that ran out ends its warp's work, raises the flag of b200sp_scaled_error and leaves rows of the output unwritten.
#pragma once

constexpr int kTileRows = 128;                      // of W: lanes of tensor memory
constexpr int kTileDepth = 128;                     // of a stage, in bytes
constexpr int kTileColsMost = 256;                  // rows of X of a tile: an accumulator's columns
constexpr int kTileWBytes = kTileRows * kTileDepth;
constexpr int kTileShared = 192 << 10;              // for stages
constexpr int kTileStagesMost = 12;
constexpr int kStoreWarps = 8, kFirstStore = 2;     // warp 0 requests, 1 multiplies, 2 ... 9 store
constexpr int kTileThreads = 32 * (kFirstStore + kStoreWarps);
// 32 x 32 results of each storing warp, of 16 bits; 32 of f32 are 128 bytes side by side as the lanes have them.
template <typename Out> constexpr int kTileStoreBytes = sizeof(Out) == 2 ? kStoreWarps * 32 * 32 * 2 : 0;
constexpr long long kTileWaitCycles = 4'000'000'000;  // two seconds
constexpr long long kTileStepCycles = 4096;           // and so many for each step of a tile, for its results

struct ScaledArgs {
    const int4 *header;      // nullptr: no experts, all rows of X by one matrix; else as in MmaArgs
    int4 mark;
    uint64_t number;
    const int *offsets;      // the experts' first rows
    int rows, experts, n, steps;
    int colsMost, box;       // rows of X of a tile at most, and of a copy
    const float *scalesX, *scalesW;
    void *y;
    long long ldy;
    int vectors;             // rows of Y start on 16 bytes
    int stages, stageBytes;
    Scalars sc;
    long long waitCycles;
    unsigned extraTx;        // 0 outside the wait test
};

__device__ int gScaledError = 0;
constexpr int kScaledWaitRanOut = 1, kScaledNoOrder = 2;

// bar: of this CTA, or with a pair of the first.
template <bool kPair> __device__ __forceinline__ void CopyTile2(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar)
{
    if constexpr (kPair)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                     "r"(x), "r"(y), "r"(bar)
                     : "memory");
}
template <bool kPair> __device__ __forceinline__ void MmaI8(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add)
{
    if constexpr (kPair)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
                     : "memory");
}

// A sum times its scales.  The product of the scales comes first, which is a normal number and leaves room for the sum if each of them lies
// between 2^-63 and 2^48 (or is 0); `plain` says that all of a warp's do.  Else the whole is taken in f64.
constexpr float kScaleLow = 0x1p-63f, kScaleHigh = 0x1p48f;
__device__ __forceinline__ bool PlainScale(float s) { return s == 0.0f || (s >= kScaleLow && s <= kScaleHigh); }
// v: sums in, results out; x: the lane's, of which sum i wants lane i's.
__device__ __forceinline__ void Scale32(float (&v)[32], float x, float w, float alpha, bool plain)
{
    if (plain) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = alpha * (__shfl_sync(0xffffffffu, x, i) * w * (float)__float_as_int(v[i]));
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            v[i] = (float)((double)alpha * ((double)__shfl_sync(0xffffffffu, x, i) * (double)w * (double)__float_as_int(v[i])));
    }
}

// Channels [f0, f0 + 128) of the expert for rows [first, first + many) of X.
struct ScaledTile {
    int expert, f0, first, many, wide, steps;  // wide: many, in whole units
};
template <bool kPair> struct ScaledTiles {
    const ScaledArgs &a;
    const int *sStart, *sOffset;  // as in Tiles
    int fTiles;
    static constexpr int kHigh = kPair ? 2 * kTileRows : kTileRows;
    static constexpr int kUnit = kPair ? 32 : 16;  // that many rows of X at least, by the shapes of kind::i8
    __device__ __forceinline__ int Count(int lo, int hi) const { return fTiles * ((hi - lo + a.colsMost - 1) / a.colsMost); }
    __device__ __forceinline__ ScaledTile At(int t) const
    {
        int lo = 0, hi = a.header != nullptr ? a.experts + 1 : 1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sStart[mid] <= t) lo = mid;
            else hi = mid;
        }
        ScaledTile m;
        m.expert = lo;
        const int within = t - sStart[lo], from = sOffset[lo], count = sOffset[lo + 1] - from;
        const int across = (count + a.colsMost - 1) / a.colsMost;
        const int per = ((count + across - 1) / across + kUnit - 1) / kUnit * kUnit;
        const int c = within % across * per;
        m.f0 = within / across * kHigh;
        m.first = from + c;
        m.many = min(per, count - c);
        m.wide = (m.many + kUnit - 1) / kUnit * kUnit;
        m.steps = lo < a.experts && m.many > 0 ? a.steps : 0;
        return m;
    }
};

template <typename Out, bool kPair>
__global__ void __launch_bounds__(kTileThreads, 1) ScaledTensorKernel(const ScaledArgs a, const __grid_constant__ CUtensorMap mapW,
                                                                      const __grid_constant__ CUtensorMap mapX)
{
    extern __shared__ unsigned char sRaw[];
    __shared__ uint64_t sFull[kTileStagesMost], sEmpty[kTileStagesMost], sDone[2], sFree[2], sLast;
    __shared__ uint32_t sTmem;
    __shared__ int sStart[kMaxExperts + 2], sOffset[kMaxExperts + 2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = kPair ? (int)(blockIdx.x & 1) : 0, first = kPair ? blockIdx.x >> 1 : blockIdx.x, step = kPair ? gridDim.x >> 1 : gridDim.x;
    const uint32_t base = (Shared(sRaw) + 1023u) & ~1023u;
    if (warp == 0) {
        if constexpr (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Shared(&sTmem)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Shared(&sTmem)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    if (tid == 0) {
        for (int s = 0; s < a.stages; ++s) {
            BarInit(sFull + s, 1);
            BarInit(sEmpty + s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            BarInit(sDone + i, 1);
            BarInit(sFree + i, kPair ? 2 * kStoreWarps : kStoreWarps);
        }
        BarInit(&sLast, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    b200sp::WaitForPrevious();
    const ScaledTiles<kPair> tiles{a, sStart, sOffset, (a.n + ScaledTiles<kPair>::kHigh - 1) / ScaledTiles<kPair>::kHigh};
    const int groups = a.header != nullptr ? a.experts + 1 : 1;
    const bool ordered = a.header == nullptr || StartsWith(a.header, a.mark, a.number);
    for (int e = tid; e <= groups; e += kTileThreads) sOffset[e] = a.header == nullptr ? e * a.rows : ordered ? __ldg(a.offsets + e) : 0;
    __syncthreads();
    if (warp == 0) {
        int run = 0;
        for (int e0 = 0; e0 <= groups; e0 += 32) {
            const int own = e0 + lane < groups ? tiles.Count(sOffset[e0 + lane], sOffset[e0 + lane + 1]) : 0;
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
    if constexpr (kPair) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sTmem;
    const int all = ordered ? sStart[groups] : 0;
    if (!ordered && tid == 0 && blockIdx.x == 0) atomicMax(&gScaledError, kScaledNoOrder);
    bool failed = false;

    if (warp == 0) {
        Ring ring;
        for (int t = first; t < all && !failed; t += step) {
            const ScaledTile m = tiles.At(t);
            const int share = kPair ? m.wide / 2 : m.wide, copies = (share + a.box - 1) / a.box;
            const int rowW = m.expert * a.n + m.f0 + rank * kTileRows, rowX = m.first + rank * share;
            for (int k = 0; k < m.steps; ++k, ring.Next(a.stages)) {
                if (ring.round > 0 && !__all_sync(0xffffffffu, BarWait(sEmpty + ring.stage, ring.Emptied(), a.waitCycles))) {
                    failed = true;
                    break;
                }
                const uint32_t at = base + ring.stage * a.stageBytes, full = kPair ? LeadersBar(sFull + ring.stage) : Shared(sFull + ring.stage);
                if (Elected()) {
                    if (rank == 0) BarExpect(sFull + ring.stage, (kPair ? 2 : 1) * (kTileWBytes + copies * a.box * kTileDepth) + a.extraTx);
                    CopyTile2<kPair>(at, &mapW, k * kTileDepth, rowW, full);
                    for (int i = 0; i < copies; ++i)
                        CopyTile2<kPair>(at + kTileWBytes + i * a.box * kTileDepth, &mapX, k * kTileDepth, rowX + i * a.box, full);
                }
                __syncwarp();
            }
        }
        if (failed && rank == 0)  // copies on their way: a bounded chance to land
            for (int i = 0; i < a.stages; ++i, ring.Next(a.stages))
                if (ring.round > 0) (void)BarWait(sFull + ring.stage, ring.Emptied(), a.waitCycles);
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t kInstr = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(ScaledTiles<kPair>::kHigh >> 4) << 24;  // signed operands, sums of 32 bits
        const bool elected = Elected();
        const uint64_t firstW = OperandAt(base, false), firstX = OperandAt(base + kTileWBytes, false);
        Ring ring;
        int tile = 0;
        for (int t = first; t < all && !failed; t += step) {
            const ScaledTile m = tiles.At(t);
            if (m.steps == 0) continue;
            const int acc = tile & 1, turn = tile >> 1;
            if (turn > 0 && !__all_sync(0xffffffffu, BarWait(sFree + acc, (uint32_t)(turn - 1) & 1u, a.waitCycles))) {
                failed = true;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t shape = kInstr | (uint32_t)(m.wide >> 3) << 17, to = tmem + acc * kTileColsMost;
            for (int k = 0; k < m.steps; ++k, ring.Next(a.stages)) {
                if (!__all_sync(0xffffffffu, BarWait(sFull + ring.stage, ring.Filled(), a.waitCycles))) {
                    failed = true;
                    break;
                }
                const uint32_t at = (uint32_t)(ring.stage * a.stageBytes) >> 4;
                if (elected) {
#pragma unroll
                    for (int i = 0; i < kTileDepth / 32; ++i) MmaI8<kPair>(to, firstW + (at + 2 * i), firstX + (at + 2 * i), shape, k > 0 || i > 0);
                    MmaCommit<kPair>(sEmpty + ring.stage);
                    if (k == m.steps - 1) MmaCommit<kPair>(sDone + acc);
                }
                __syncwarp();
            }
            ++tile;
        }
        if (elected) MmaCommit<kPair>(&sLast);  // when every product started here is complete, also after a failure
        __syncwarp();
        (void)BarWait(&sLast, 0, a.waitCycles);
    } else if (warp >= kFirstStore) {
        const int quarter = warp & 3, half = (warp - kFirstStore) >> 2;  // the lanes of tensor memory that the warp may read; every other 32 columns
        const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
        Out *const sOut = reinterpret_cast<Out *>(sRaw + (base - Shared(sRaw)) + a.stages * a.stageBytes) + (warp - kFirstStore) * 1024;
        Out *const out = static_cast<Out *>(a.y);
        int tile = 0;
        for (int t = first; t < all; t += step) {
            const ScaledTile m = tiles.At(t);
            const int f0 = m.f0 + rank * kTileRows + quarter * 32;  // the warp's 32 channels
            const bool in = f0 + lane < a.n;
            // what the results are scaled by is asked for before they are waited for
            const float w = m.steps > 0 && in ? __ldg(a.scalesW + (long long)m.expert * a.n + f0 + lane) : 0.0f;
            float scales[kTileColsMost / 64];
#pragma unroll
            for (int i = 0; i < kTileColsMost / 64; ++i) {
                const int c = half * 32 + 64 * i + lane;
                scales[i] = m.steps > 0 && c < m.many ? __ldg(a.scalesX + m.first + c) : 0.0f;
            }
            const int acc = tile & 1, turn = tile >> 1;
            if (m.steps > 0) {
                if (!BarWaitWarp(sDone + acc, (uint32_t)turn & 1u, a.waitCycles + m.steps * kTileStepCycles)) {
                    failed = true;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                ++tile;
            }
            const uint32_t from = tmem + ((uint32_t)quarter << 21) + acc * kTileColsMost;
            for (int c0 = half * 32; c0 < m.many; c0 += 64) {
                float v[32] = {};
                const float x = scales[0];
#pragma unroll
                for (int i = 1; i < kTileColsMost / 64; ++i) scales[i - 1] = scales[i];
                if (m.steps > 0) {
                    LoadColumns32(from + c0, v);
                    Scale32(v, x, w, alpha, __all_sync(0xffffffffu, PlainScale(w) && PlainScale(x)));
                }
                const int live = min(32, m.many - c0);
                Out *const to = out + (long long)(m.first + c0) * a.ldy + f0;
                if (sizeof(Out) == 2 && a.vectors && beta == 0.0f) {
                    if constexpr (sizeof(Out) == 2) {
                        // Through shared memory, so that 16 bytes of a row are stored at once and a row's 32 channels side by side.
                        constexpr int kN = 16 / (int)sizeof(Out), kPieces = 32 / kN;
#pragma unroll
                        for (int i = 0; i < 32; ++i) sOut[32 * i + lane] = FromFloat<Out>(v[i]);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            const int c = (32 * i + lane) / kPieces, at = lane % kPieces * kN;
                            const uint4 piece = *reinterpret_cast<const uint4 *>(sOut + 32 * c + at);
                            Out *const row = to + c * a.ldy + at;
                            if (c < live && f0 + at + kN <= a.n) *reinterpret_cast<uint4 *>(row) = piece;
                            else if (c < live)  // the last channels
                                for (int j = 0; f0 + at + j < a.n; ++j) row[j] = sOut[32 * c + at + j];
                        }
                        __syncwarp();
                    }
                } else {
                    // A channel a lane.  What is read is asked for before anything is stored.
#pragma unroll
                    for (int g = 0; g < 32; g += 8) {
                        float old[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) old[i] = beta != 0.0f && in && g + i < live ? ToFloat(to[(g + i) * a.ldy + lane]) : 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float u = beta != 0.0f ? fmaf(beta, old[i], v[g + i]) : v[g + i];
                            if (in && g + i < live) to[(g + i) * a.ldy + lane] = FromFloat<Out>(u);
                        }
                    }
                }
            }
            if (m.steps > 0) {  // all that this warp reads of the accumulator
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) BarArriveAt(kPair ? LeadersBar(sFree + acc) : Shared(sFree + acc));
            }
        }
    }
    __syncwarp();
    if (failed) atomicMax(&gScaledError, kScaledWaitRanOut);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // The other CTA may still signal barriers here, and the pair's tensor memory is freed by both.
    if constexpr (kPair) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 0) {
        if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------- host

// Rows of bytes, `high` of them by 128, swizzled; what is past the last column or row arrives as zeros.
inline bool MapOfBytes(CUtensorMap *map, const void *at, long long cols, long long rows, long long ld, int high)
{
    const EncodeTiled encode = Encoder();
    if (encode == nullptr) return false;
    const cuuint64_t size[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {kTileDepth, (cuuint32_t)high}, step[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(at), size, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

long long gScaledWaitCycles = kTileWaitCycles;
unsigned gScaledExtraTx = 0;

template <typename Out, bool kPair>
cudaError_t LaunchScaled(ScaledArgs a, const CUtensorMap &mapW, const CUtensorMap &mapX, cudaStream_t stream)
{
    a.stageBytes = kTileWBytes + a.colsMost * kTileDepth / (kPair ? 2 : 1);
    a.stages = std::min(kTileShared / a.stageBytes, kTileStagesMost);
    a.waitCycles = gScaledWaitCycles;
    a.extraTx = gScaledExtraTx;
    const cudaError_t e = AllowShared<ScaledTensorKernel<Out, kPair>>(kTileShared + kTileStoreBytes<Out> + 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(b200sp_sm_count() / 2 * 2));
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = (size_t)(a.stages * a.stageBytes + kTileStoreBytes<Out> + 1024);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kPair ? 2 : 1;
    b200sp_note_launches(1);
    return cudaLaunchKernelEx(&cfg, ScaledTensorKernel<Out, kPair>, a, mapW, mapX);
}
