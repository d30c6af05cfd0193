// Products in 8-bit integers on the tensor cores: included by scaled.cu.
//
// Y^T = W X^T: a tile is 128 channels (rows of W, the rows "M" of tcgen05.mma, kind::i8) by up to 256 rows of X (its "N"), so that with few rows, as
// when single tokens are served, N shrinks and what moves is W.  With experts, whose rows lie side by side, a tile is one expert's.
// One warp requests both operands by TMA, in rows of 128 bytes, swizzled; one starts the products; eight empty the accumulators, of which there are
// two: the next tile is summed meanwhile.  Sums are whole numbers of 32 bits; they are scaled in f32 and rounded once.
// Many rows go to pairs of CTAs on tiles of 256 channels, which read half as much of X; few tiles to clusters that share their steps (ScaledSplitKernel); few rows
// to warps without tiles (ScaledFewKernel).  FormOf decides.
// What bounds it: with many rows the tensor cores (67 % of the cycles) and what a step asks of shared memory and L2 (32 KB a CTA in some 650 clocks, of which its
// products take 512), in long runs the power cap; with short sums the storing of the results (8000 clocks a tile; one of 16 steps takes 16,500 in all, as much as
// its products and that together).  One B200: 8192 x 4096 by 4096 bf16 out 97 us (2.8 POPS), 8192 x 4096 by 8192 183 alone and 220 in runs of seconds, 32,768 x 2048
// by 2048 115; the rows of 8192 tokens, four of 32 experts, 2048 x 2048 126. By single CTAs on tiles of 128 channels: 5 to 10 % longer.  Results stored 64 bytes of
// a row at a time by two bytes a lane: twice as long as 16 a lane.
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
// 32 rows of Y by 128 channels, of 16 bits, of each half of the storing warps; 32 of f32 are 128 bytes side by side as the lanes have them.
template <typename Out> constexpr int kTileStoreBytes = sizeof(Out) == 2 ? 2 * 32 * kTileRows * 2 : 0;
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
    int split, tmemColumns;  // of ScaledSplitKernel
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
// The four warps of a half of a tile's columns.
__device__ __forceinline__ void StoreBarrier(int half)
{
    __syncwarp();
    asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
}
// Whether a wait ran out for none of them: they go on together, or not at all.
__device__ __forceinline__ bool StoreAgree(int half, bool ok)
{
    uint32_t all;
    __syncwarp();
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(all)
                 : "r"((uint32_t)ok), "r"(1 + half)
                 : "memory");
    return all != 0;
}

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

// The experts' first rows (and that of the group of no expert; without experts there is one group of all rows), and the first of the units of work,
// `count` of a number of rows, of each.  By a whole CTA, synchronised when the first are there, of which warp 0 is the last.  False without an order.
template <typename Count>
__device__ __forceinline__ bool WorkTable(const ScaledArgs &a, int groups, int threads, int *sStart, int *sOffset, Count &&count)
{
    const int tid = threadIdx.x, lane = tid & 31;
    const bool ordered = a.header == nullptr || StartsWith(a.header, a.mark, a.number);
    for (int e = tid; e <= groups; e += threads) sOffset[e] = a.header == nullptr ? e * a.rows : ordered ? __ldg(a.offsets + e) : 0;
    __syncthreads();
    if (tid < 32) {
        int run = 0;
        for (int e0 = 0; e0 <= groups; e0 += 32) {
            const int own = e0 + lane < groups ? count(sOffset[e0 + lane + 1] - sOffset[e0 + lane]) : 0;
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
    return ordered;
}
// The group that a unit of work is of.
__device__ __forceinline__ int GroupOf(const int *sStart, int groups, int unit)
{
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sStart[mid] <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ float Scaled(int sum, float x, float w, float alpha)
{
    return PlainScale(w) && PlainScale(x) ? alpha * (x * w * (float)sum) : (float)((double)alpha * ((double)x * (double)w * (double)sum));
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
    __device__ __forceinline__ int Count(int rows) const { return fTiles * ((rows + a.colsMost - 1) / a.colsMost); }
    __device__ __forceinline__ ScaledTile At(int t) const
    {
        const int lo = GroupOf(sStart, a.header != nullptr ? a.experts + 1 : 1, t);
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
    const bool ordered = WorkTable(a, groups, kTileThreads, sStart, sOffset, [&](int count) { return tiles.Count(count); });
    TensorBefore();
    __syncthreads();
    if constexpr (kPair) ClusterMeet();
    TensorAfter();
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
            TensorAfter();
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
    } else if (warp >= kFirstStore) {
        const int quarter = warp & 3, half = (warp - kFirstStore) >> 2;  // the lanes of tensor memory that the warp may read; every other 32 columns
        const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
        Out *const sOut = reinterpret_cast<Out *>(sRaw + (base - Shared(sRaw)) + a.stages * a.stageBytes) + half * (32 * kTileRows);
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
                if (!StoreAgree(half, BarWaitWarp(sDone + acc, (uint32_t)turn & 1u, a.waitCycles + m.steps * kTileStepCycles))) {
                    failed = true;
                    break;
                }
                TensorAfter();
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
                        // Through shared memory, where the four warps of these columns meet, so that 256 bytes of a row are stored side by side.
#pragma unroll
                        for (int i = 0; i < 32; ++i) sOut[kTileRows * i + quarter * 32 + lane] = FromFloat<Out>(v[i]);
                        StoreBarrier(half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c = quarter * 8 + 2 * i + (lane >> 4), at = (lane & 15) * 8, channel = f0 - quarter * 32 + at;
                            const uint4 piece = *reinterpret_cast<const uint4 *>(sOut + kTileRows * c + at);
                            Out *const row = to + c * a.ldy - quarter * 32 + at;
                            if (c < live && channel + 8 <= a.n) *reinterpret_cast<uint4 *>(row) = piece;
                            else if (c < live)  // the last channels
                                for (int j = 0; channel + j < a.n; ++j) row[j] = sOut[kTileRows * c + at + j];
                        }
                        StoreBarrier(half);
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
                TensorBefore();
                __syncwarp();
                if (lane == 0) BarArriveAt(kPair ? LeadersBar(sFree + acc) : Shared(sFree + acc));
            }
        }
    }
    __syncwarp();
    if (failed) atomicMax(&gScaledError, kScaledWaitRanOut);
    TensorBefore();
    __syncthreads();
    // Every product has ended, and in a pair the last signal of the first CTA's commits has come in at the other one, too, before either of them ends.
    if (warp == 0) (void)BarWaitWarp(&sLast, 0, a.waitCycles);
    // The other CTA may still signal barriers here, and the pair's tensor memory is freed by both.
    if constexpr (kPair) ClusterMeet();
    TensorAfter();
    if (warp == 0) {
        if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Few tiles, as when some tokens are served: the CTAs of a cluster share the steps of one tile, and each adds up a part of its columns from
// all their accumulators, through shared memory.  Sums of whole numbers may be regrouped.  61 rows of 4096 by 4096: 11.2 us, 14.4 by whole tiles; 61 of 2040 by
// 1111 7.1 and 9.5.  What bounds it is latency: a launch, its ends and two meetings of the cluster are 5 us.
constexpr int kSplitThreads = 256, kSplitMost = 8;  // CTAs of a cluster: the portable most
// At least so much shared memory, which leaves no room for another CTA that takes tensor memory, of this library or any other, and fills shared memory with tiles for
// it.  Clusters (and pairs) of two streams that each wait for the tensor memory of the other would wait for ever.  (It costs nothing: FormOf takes no more clusters
// than have SMs of their own.)
constexpr int kSplitShared = kTileShared;

__device__ __forceinline__ int LoadRemote(uint32_t at, int rank)
{
    uint32_t there;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(there) : "memory");
    return v;
}

template <typename Out>
__global__ void __launch_bounds__(kSplitThreads, 1) ScaledSplitKernel(const ScaledArgs a, const __grid_constant__ CUtensorMap mapW,
                                                                      const __grid_constant__ CUtensorMap mapX)
{
    extern __shared__ unsigned char sRaw[];
    __shared__ uint64_t sFull[kTileStagesMost], sEmpty[kTileStagesMost], sDone;
    __shared__ uint32_t sTmem;
    __shared__ int sFailed;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int split = a.split, rank = (int)(blockIdx.x % split), tile = (int)(blockIdx.x / split);
    const uint32_t base = (Shared(sRaw) + 1023u) & ~1023u;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Shared(&sTmem)), "r"(a.tmemColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 32) {
        for (int s = 0; s < a.stages; ++s) {
            BarInit(sFull + s, 1);
            BarInit(sEmpty + s, 1);
        }
        BarInit(&sDone, 1);
        sFailed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    b200sp::WaitForPrevious();
    TensorBefore();
    __syncthreads();
    TensorAfter();
    const uint32_t tmem = sTmem;
    // Tiles side by side along the rows of X first.
    const int across = (a.rows + a.colsMost - 1) / a.colsMost, f0 = tile / across * kTileRows, first = tile % across * a.colsMost;
    const int many = min(a.colsMost, a.rows - first), wide = (many + 15) / 16 * 16;
    const int from = (int)((long long)a.steps * rank / split), to = (int)((long long)a.steps * (rank + 1) / split);
    bool failed = false;
    if (warp == 0) {
        Ring ring;
        const int copies = (wide + a.box - 1) / a.box;
        for (int k = from; k < to; ++k, ring.Next(a.stages)) {
            if (ring.round > 0 && !__all_sync(0xffffffffu, BarWait(sEmpty + ring.stage, ring.Emptied(), a.waitCycles))) {
                failed = true;
                break;
            }
            const uint32_t at = base + ring.stage * a.stageBytes, full = Shared(sFull + ring.stage);
            if (Elected()) {
                BarExpect(sFull + ring.stage, kTileWBytes + copies * a.box * kTileDepth + a.extraTx);
                CopyTile2<false>(at, &mapW, k * kTileDepth, f0, full);
                for (int i = 0; i < copies; ++i)
                    CopyTile2<false>(at + kTileWBytes + i * a.box * kTileDepth, &mapX, k * kTileDepth, first + i * a.box, full);
            }
            __syncwarp();
        }
        if (failed)  // copies on their way: a bounded chance to land
            for (int i = 0; i < a.stages; ++i, ring.Next(a.stages))
                if (ring.round > 0) (void)BarWait(sFull + ring.stage, ring.Emptied(), a.waitCycles);
    } else if (warp == 1) {
        const uint32_t shape = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(wide >> 3) << 17 | (uint32_t)(kTileRows >> 4) << 24;
        const bool elected = Elected();
        const uint64_t firstW = OperandAt(base, false), firstX = OperandAt(base + kTileWBytes, false);
        Ring ring;
        for (int k = from; k < to; ++k, ring.Next(a.stages)) {
            if (!__all_sync(0xffffffffu, BarWait(sFull + ring.stage, ring.Filled(), a.waitCycles))) {
                failed = true;
                break;
            }
            const uint32_t at = (uint32_t)(ring.stage * a.stageBytes) >> 4;
            if (elected) {
#pragma unroll
                for (int i = 0; i < kTileDepth / 32; ++i) MmaI8<false>(tmem, firstW + (at + 2 * i), firstX + (at + 2 * i), shape, k > from || i > 0);
                MmaCommit<false>(sEmpty + ring.stage);
            }
            __syncwarp();
        }
        if (elected) MmaCommit<false>(&sDone);  // when every product started here is complete, also after a failure
    }
    __syncwarp();
    if (!BarWaitWarp(&sDone, 0, 2 * a.waitCycles + (to - from) * kTileStepCycles)) failed = true;  // longer than the waits above
    if (failed) sFailed = 1;
    TensorAfter();
    __syncthreads();
    // The sums, a column of 128 channels after the other, where the stages were.
    const int quarter = warp & 3;
    if (sFailed == 0) {
        for (int c0 = (warp >> 2) * 32; c0 < wide; c0 += 64) {
            float v[32];
            LoadColumns32(tmem + ((uint32_t)quarter << 21) + c0, v);
            int *const sums = reinterpret_cast<int *>(sRaw + (base - Shared(sRaw))) + c0 * kTileRows + quarter * 32 + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (c0 + i < wide) sums[i * kTileRows] = __float_as_int(v[i]);
        }
    }
    TensorBefore();  // all that is read of tensor memory
    ClusterMeet();
    int bad = 0;
    for (int r = 0; r < split; ++r) bad |= LoadRemote(Shared(&sFailed), r);
    if (bad == 0) {
        const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
        const int f = tid & (kTileRows - 1), channel = f0 + f;
        const bool in = channel < a.n;
        const float w = in ? __ldg(a.scalesW + channel) : 0.0f;
        constexpr int kTogether = 4;  // columns whose sums are asked for at once
        for (int c0 = rank * 2 + (tid >> 7); c0 < many; c0 += 2 * split * kTogether) {
            int sum[kTogether] = {};
            float x[kTogether], old[kTogether];
#pragma unroll
            for (int u = 0; u < kTogether; ++u) {
                const int c = min(c0 + 2 * split * u, many - 1);
                const uint32_t at = base + (c * kTileRows + f) * 4;
                for (int r = 0; r < split; ++r) sum[u] += LoadRemote(at, r);
                x[u] = __ldg(a.scalesX + first + c);
                old[u] = beta != 0.0f && in ? ToFloat(static_cast<const Out *>(a.y)[(long long)(first + c) * a.ldy + channel]) : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < kTogether; ++u) {
                const int c = c0 + 2 * split * u;
                const float v = Scaled(sum[u], x[u], w, alpha);
                if (in && c < many)
                    static_cast<Out *>(a.y)[(long long)(first + c) * a.ldy + channel] = FromFloat<Out>(beta != 0.0f ? fmaf(beta, old[u], v) : v);
            }
        }
    } else if (rank == 0 && tid == 0) {
        atomicMax(&gScaledError, kScaledWaitRanOut);
    }
    // The others may still read this CTA's sums.
    ClusterMeet();
    TensorAfter();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmemColumns) : "memory");
}

// Few rows at a matrix: no tile, but warps at two rows of W and of X.  What moves is W, in pieces of 512 bytes of a row, of which a warp asks for eight at
// once; rows of X come from L1.  Products of four bytes at a time (dp4a).  With `parts` > 1 so many warps share an item's columns.
// One row of 4096 by 4096: 6.6 us with the matrix from DRAM, 4.7 from L2; 2.5 are a launch and its ends, 2.6 the matrix at the copy rate.  Other shapes, rows of X x
// of W, pieces: 1 x 2, 8 9.3 us, 1 x 4, 4 8.4, 2 x 4, 2 8.6.  Eight rows of X are bound by the rate of dp4a, some 10 lanes a clock and SM: 19 us; by the int8
// products of a warp (mma.sync) 10.3, but one row 8.6, and small matrices half as long again.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32, kFewPiece = 512, kFewRowsX = 2;

template <typename Out>
__global__ void __launch_bounds__(kFewThreads) ScaledFewKernel(const ScaledArgs a, const int8_t *__restrict__ matX, long long ldx,
                                                               const int8_t *__restrict__ matW, long long ldw, int depth, int parts)
{
    constexpr int kM = kFewRowsX, kR = 2, kAhead = 4;
    __shared__ int sStart[kMaxExperts + 2], sOffset[kMaxExperts + 2];
    __shared__ int sPart[2][kFewWarps][kM * kR];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    b200sp::WaitForPrevious();
    const int groups = a.header != nullptr ? a.experts + 1 : 1, perRow = (a.n + kR - 1) / kR;
    const bool ordered = WorkTable(a, groups, kFewThreads, sStart, sOffset, [&](int rows) { return (rows + kM - 1) / kM * perRow; });
    __syncthreads();
    if (!ordered) {
        if (tid == 0 && blockIdx.x == 0) atomicMax(&gScaledError, kScaledNoOrder);
        return;
    }
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
    const int all = sStart[groups], side = kFewWarps / parts, part = warp % parts;
    const int pieces = depth / 16, rest = depth % 16;  // of 16 bytes
    int turn = 0;
    for (long long item = (long long)blockIdx.x * side + warp / parts; item < all; item += (long long)gridDim.x * side, turn ^= 1) {
        const int expert = GroupOf(sStart, groups, (int)item), within = (int)item - sStart[expert];
        const int chunk = within / perRow, f0 = (within - chunk * perRow) * kR;
        const int first = sOffset[expert] + chunk * kM, many = min(kM, sOffset[expert + 1] - first);
        const bool live = expert < a.experts;
        int sum[kR][kM] = {};
        if (live) {
            const int8_t *w[kR];
#pragma unroll
            for (int r = 0; r < kR; ++r) w[r] = matW + ((long long)expert * a.n + min(f0 + r, a.n - 1)) * ldw;
            const int8_t *const x = matX + first * ldx;
            for (int p0 = part * 32 + lane; p0 < pieces; p0 += parts * 32 * kAhead) {
                int4 v[kAhead][kR];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int p = p0 + u * parts * 32;
#pragma unroll
                    for (int r = 0; r < kR; ++r)
                        v[u][r] = p < pieces ? __ldg(reinterpret_cast<const int4 *>(w[r]) + p) : make_int4(0, 0, 0, 0);
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int p = min(p0 + u * parts * 32, pieces - 1);
#pragma unroll
                    for (int m = 0; m < kM; ++m) {
                        if (m >= many) break;
                        const int4 y = __ldg(reinterpret_cast<const int4 *>(x + m * ldx) + p);
#pragma unroll
                        for (int r = 0; r < kR; ++r)
                            sum[r][m] = __dp4a(v[u][r].w, y.w, __dp4a(v[u][r].z, y.z, __dp4a(v[u][r].y, y.y, __dp4a(v[u][r].x, y.x, sum[r][m]))));
                    }
                }
            }
            if (part == 0 && lane < rest) {  // the last columns, which are no whole piece
                const int c = pieces * 16 + lane;
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    if (m >= many) break;
#pragma unroll
                    for (int r = 0; r < kR; ++r) sum[r][m] += (int)w[r][c] * (int)x[m * ldx + c];
                }
            }
        }
        int mine = 0;  // of lane m * kR + r: the sum of row m and channel r
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                const int total = __reduce_add_sync(0xffffffffu, sum[r][m]);
                if (lane == m * kR + r) mine = total;
            }
        if (parts > 1) {  // two places in turn: one is written while others may still read the other
            if (lane < kM * kR) sPart[turn][warp][lane] = mine;
            __syncwarp();
            asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / parts), "r"(32 * parts) : "memory");
            if (part != 0) continue;
            mine = 0;
            if (lane < kM * kR)
                for (int i = 0; i < parts; ++i) mine += sPart[turn][warp + i][lane];
        }
        const int m = lane / kR, f = f0 + lane % kR;
        if (m >= many || f >= a.n) continue;
        float v = 0.0f;
        if (live) v = Scaled(mine, __ldg(a.scalesX + first + m), __ldg(a.scalesW + (long long)expert * a.n + f), alpha);
        Out *const to = static_cast<Out *>(a.y) + (first + m) * a.ldy + f;
        *to = FromFloat<Out>(beta != 0.0f ? fmaf(beta, ToFloat(*to), v) : v);
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

template <typename Out> cudaError_t LaunchSplit(ScaledArgs a, const CUtensorMap &mapW, const CUtensorMap &mapX, cudaStream_t stream)
{
    a.stageBytes = kTileWBytes + a.colsMost * kTileDepth;
    a.stages = std::min({kTileShared / a.stageBytes, kTileStagesMost, (a.steps + a.split - 1) / a.split});
    a.tmemColumns = std::max(32, a.colsMost);
    a.waitCycles = gScaledWaitCycles;
    a.extraTx = gScaledExtraTx;
    const cudaError_t e = AllowShared<ScaledSplitKernel<Out>>(kTileShared + 1024);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)((a.n + kTileRows - 1) / kTileRows) * ((a.rows + a.colsMost - 1) / a.colsMost);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * a.split));
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = (size_t)(std::max({a.stages * a.stageBytes, a.colsMost * kTileRows * 4, kSplitShared}) + 1024);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    b200sp_note_launches(1);
    return cudaLaunchKernelEx(&cfg, ScaledSplitKernel<Out>, a, mapW, mapX);
}

// chunks: of two rows of X, at most.
template <typename Out>
cudaError_t LaunchFew(const ScaledArgs &a, const void *x, long long ldx, const void *w, long long ldw, int depth, long long chunks, cudaStream_t stream)
{
    // Warps for all SMs: items that are fewer are shared, as long as a warp has columns of its own.
    const long long items = (a.n + 1) / 2 * chunks, warps = (long long)b200sp_sm_count() * 24;
    int parts = 1;
    while (parts < kFewWarps && items * parts < warps && depth > parts * kFewPiece) parts *= 2;
    const long long ctas = (items * parts + kFewWarps - 1) / kFewWarps;
    b200sp_note_launches(1);
    return b200sp::LaunchChained(ScaledFewKernel<Out>, (unsigned)std::min(ctas, (long long)b200sp_sm_count() * 4), kFewThreads, 0, stream, a,
                                 static_cast<const int8_t *>(x), ldx, static_cast<const int8_t *>(w), ldw, depth, parts);
}
