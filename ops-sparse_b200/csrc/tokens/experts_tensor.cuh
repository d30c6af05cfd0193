// The experts' products on the tensor cores: included by experts.cu.
//
// A tile is 128 columns of Y (of an expert's matrix, the rows "M" of tcgen05.mma) by up to 256 entries of the expert (its "N"),
// that is Y^T = op(W) X^T: with few entries, as when single tokens are served, N shrinks to 16 and what moves is W,
// at full width; the accumulator's lanes are then columns of Y, and a store is 32 of them for one entry.
// The gradient's tile is 128 rows of dW by up to 256 of its columns, summed over the expert's entries.
//
// One CTA per SM, or a pair of CTAs on tiles twice as high, walks over the tiles of all experts.  One warp requests W by TMA; twelve gather
// the rows of X (and dY), which may lie anywhere, by cp.async, so that nothing is laid out in between; one starts the products, four
// empty the accumulators, of which there are two: the next tile is summed meanwhile.
// What bounds it: with many entries the tensor cores (71 % of the cycles) and what comes from L2, 32 KB a step and SM at some 58 bytes a clock,
// where the products of a step take 450; with few the weights, once from DRAM.  One B200: 8192 tokens, four of 32 experts, 2048 x 2048, bf16
// (275 GFLOP) 233 us in runs of milliseconds, 274 in runs of seconds under the power cap; 16 tokens, 8 of 64 experts, 2048 x 1024 41 us
// (0.9 of the copy rate).  The same by rows of X from TMA
// (tile::gather4: 18 clocks a row of 128 bytes and SM) 1250, by one CTA a tile 380.
// Operands arrive in rows of 128 bytes, swizzled: K-major where those run along the sum (X; W with opW = T), MN-major
// where they run along the tile (W with opW = N; both of the gradient's).
//
// Every wait is bounded, that for a tile's results by its steps.  One that ran out ends its warp's work, raises the flag of b200sp_experts_error and leaves rows of the
// output unwritten; nothing waits for ever, and tensor memory is freed when copies and products in flight have had time to
// land.
#pragma once

#include <cuda.h>

constexpr int kMmaRows = 128;                      // of a tile: lanes of tensor memory
constexpr int kMmaDepth = 64;                      // of a stage: 128 bytes
constexpr int kMmaColsMost = 256;                  // of a tile: an accumulator's columns
constexpr int kMmaABytes = kMmaRows * kMmaDepth * 2;
constexpr int kMmaBlockBytes = kMmaDepth * 128;    // MN-major: 64 rows along the sum, 64 elements along the tile
constexpr int kMmaShared = 192 << 10;              // for stages
constexpr int kMmaStagesMost = 12;
template <typename Out> constexpr int kMmaStoreBytes = 4 * 32 * 32 * (int)sizeof(Out);  // 32 x 32 results of each storing warp
constexpr int kMmaGatherWarps = 12, kMmaPartsMost = 2;  // warps that gather, of them at a stage
constexpr int kMmaFirstGather = 6;                 // warp 0 requests W, 1 multiplies, 2 ... 5 store, 6 ... gather
constexpr int kMmaThreads = 32 * (kMmaFirstGather + kMmaGatherWarps);
constexpr long long kMmaWaitCycles = 4'000'000'000;  // two seconds
// A tile's results may take longer, by its steps: all SMs at once ask DRAM for 48 KB a step, some 2000 clocks, where nothing comes from L2.
constexpr long long kMmaStepCycles = 4096;

enum class Mode { kProductT, kProductN, kGrad };

struct MmaArgs {
    const int4 *header;    // has to be `mark`, and `number` unless that is 0, or nothing of the rest is looked at
    int4 mark;
    uint64_t number;
    const int *offsets, *entries, *rows;
    void *out;
    long long ldo;
    int experts, n, d;
    int byEntry;
    const void *dy, *x;
    long long ldy, ldx;
    int vectors;           // rows of the output start on 16 bytes
    int colsMost;          // of a tile
    int stages, stageBytes;
    int parts;             // warps that gather a stage
    Scalars sc;
    long long waitCycles;
    unsigned extraTx;      // 0 outside the wait test: bytes that W's barrier expects beyond those copied; gathering threads do not arrive
};

__device__ int gExpertsError = 0;
constexpr int kWaitRanOut = 1, kNoOrder = 2;

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
    const uint64_t leading = alongTile ? kMmaBlockBytes >> 4 : 1, stride = 1024 >> 4;
    return (uint64_t)((at & 0x3ffff) >> 4) | leading << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}
template <bool kPair> __device__ __forceinline__ void Mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add)
{
    if constexpr (kPair)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
                     : "memory");
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

// What a tile is: columns [f0, f0 + 128) of Y for entries [first, first + many) of the expert, or rows [f0, ...) and columns
// [first, first + many) of its gradient.
struct MmaTile {
    int expert, f0, first, many, wide, steps;  // wide: many, in whole units
};

template <Mode kMode, bool kPair> struct Tiles {
    const MmaArgs &a;
    const int *sStart;   // [experts + 2]: the first tile of every expert, and of the group of no expert
    const int *sOffset;  // [experts + 2]: their first entries
    int fTiles;
    static constexpr int kHigh = kPair ? 2 * kMmaRows : kMmaRows;
    // Products take entries by sixteens, gradients whole blocks of 64 columns, for each CTA of a pair.
    static constexpr int kUnit = kMode != Mode::kGrad ? 16 : kPair ? 128 : 64;

    __device__ __forceinline__ int Groups() const { return kMode == Mode::kGrad ? a.experts : a.experts + 1; }
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
        const int within = t - sStart[lo], from = sOffset[lo], count = sOffset[lo + 1] - from;
        const int length = kMode == Mode::kGrad ? a.d : count;
        const int across = (length + a.colsMost - 1) / a.colsMost;
        const int per = ((length + across - 1) / across + kUnit - 1) / kUnit * kUnit;
        const int c = within % across * per;
        m.f0 = within / across * kHigh;
        m.first = kMode == Mode::kGrad ? c : from + c;
        m.many = min(per, length - c);
        m.wide = (m.many + kUnit - 1) / kUnit * kUnit;
        if (kMode == Mode::kGrad) m.steps = (count + kMmaDepth - 1) / kMmaDepth;
        else m.steps = lo < a.experts && m.many > 0 ? ((kMode == Mode::kProductT ? a.d : a.n) + kMmaDepth - 1) / kMmaDepth : 0;
        return m;
    }
};

template <typename T, typename Out, Mode kMode, bool kPair>
__global__ void __launch_bounds__(kMmaThreads, 1) ExpertsTensorKernel(const MmaArgs a, const __grid_constant__ CUtensorMap mapW)
{
    extern __shared__ unsigned char sRaw[];
    __shared__ uint64_t sFull[kMmaStagesMost], sEmpty[kMmaStagesMost], sDone[2], sFree[2], sLast;
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
            BarInit(sFull + s, (kMode != Mode::kGrad) + a.parts * (kPair ? 2 : 1));  // W's request, the gathering warps of every CTA
            BarInit(sEmpty + s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            BarInit(sDone + i, 1);
            BarInit(sFree + i, kPair ? 8 : 4);
        }
        BarInit(&sLast, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    b200sp::WaitForPrevious();
    const Tiles<kMode, kPair> tiles{a, sStart, sOffset,
                                    ((kMode == Mode::kProductN ? a.d : a.n) + Tiles<kMode, kPair>::kHigh - 1) / Tiles<kMode, kPair>::kHigh};
    const int groups = tiles.Groups();
    const int4 found = __ldg(a.header);
    const bool ordered = found.x == a.mark.x && found.y == a.mark.y && found.z == a.mark.z && found.w == a.mark.w &&
                         (a.number == 0 || __ldg(reinterpret_cast<const unsigned long long *>(a.header + 1)) == a.number);
    for (int e = tid; e <= groups; e += kMmaThreads) sOffset[e] = ordered ? __ldg(a.offsets + e) : 0;
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
    if (!ordered && tid == 0 && blockIdx.x == 0) atomicMax(&gExpertsError, kNoOrder);
    bool failed = false;

    if (kMode != Mode::kGrad && warp == 0) {
        Ring ring;
        for (int t = first; t < all && !failed; t += step) {
            const MmaTile m = tiles.At(t);
            const int f0 = m.f0 + rank * kMmaRows;
            for (int k = 0; k < m.steps; ++k, ring.Next(a.stages)) {
                if (ring.round > 0 && !__all_sync(0xffffffffu, BarWait(sEmpty + ring.stage, ring.Emptied(), a.waitCycles))) {
                    failed = true;
                    break;
                }
                const uint32_t at = base + ring.stage * a.stageBytes, full = kPair ? LeadersBar(sFull + ring.stage) : Shared(sFull + ring.stage);
                if (Elected()) {
                    if (rank == 0) BarExpect(sFull + ring.stage, (kPair ? 2 : 1) * kMmaABytes + a.extraTx);
                    if (kMode == Mode::kProductT) {
                        CopyTile3<kPair>(at, &mapW, k * kMmaDepth, f0, m.expert, full);
                    } else {
                        CopyTile3<kPair>(at, &mapW, f0, k * kMmaDepth, m.expert, full);
                        CopyTile3<kPair>(at + kMmaBlockBytes, &mapW, f0 + 64, k * kMmaDepth, m.expert, full);
                    }
                }
                __syncwarp();
            }
        }
        if (failed && rank == 0)  // copies on their way: a bounded chance to land
            for (int i = 0; i < a.stages; ++i, ring.Next(a.stages))
                if (ring.round > 0) (void)BarWait(sFull + ring.stage, ring.Emptied(), a.waitCycles);
    } else if (warp >= kMmaFirstGather && warp < kMmaFirstGather + a.parts * a.stages) {
        // Stages are the warps' in turn, one's or a pair of warps': they ask for all of its rows, wait for them and say so, while the others are
        // at the stages beside it.  No more turns than stages: whoever is at stage q knows that q - stages has been used up, so that the
        // wait for q + turns - stages can not be answered by the round before it.  (All warps at every stage, a share each, and an arrival
        // of every thread: a stage's round took 2900 clocks without any copy.)
        // Eight lanes side by side on 128 bytes of a row: lane l has piece l % 8 of rows l / 8, l / 8 + 4, ...
        const int mine = (warp - kMmaFirstGather) / a.parts, part = (warp - kMmaFirstGather) % a.parts;
        const int warps = min(kMmaGatherWarps / a.parts, a.stages), piece = lane & 7, high = lane >> 3;
        const uint32_t place = base + high * 128;
        const uint32_t even = (uint32_t)(piece ^ high) << 4, odd = (uint32_t)(piece ^ (high + 4)) << 4;  // swizzled: rows high, high + 4 of eight
        Ring ring;
        ring.On(mine, a.stages);
        auto free = [&]() { return ring.round == 0 || BarWaitWarp(sEmpty + ring.stage, ring.Emptied(), a.waitCycles); };
        auto asked = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor cores read it from here on
            __syncwarp();
            if (lane == 0 && a.extraTx == 0) BarArriveAt(LeadersBar(sFull + ring.stage));
            ring.On(warps, a.stages);
        };
        int turn = mine;  // steps until the next of this warp's stages
        if constexpr (kMode != Mode::kGrad) {
            constexpr int kRows = kMmaColsMost / (kPair ? 2 : 1) / 32 / kMmaPartsMost;  // times 32
            const int depth = kMode == Mode::kProductT ? a.d : a.n;
            const int *const rowOf = a.byEntry ? a.entries : a.rows;
            const char *const x = static_cast<const char *>(a.x);
            const uint32_t pitch = (uint32_t)a.ldx * 2;
            // Eights of rows belong to the parts in turn: the lane's own, of which it knows the places, are row 8 * (part + parts * e)
            // + lane % 8 with e = lane / 8, lane / 8 + 4, ...  (What is past the last entry is a copy of row 0, of whose sums nobody asks.)
            uint32_t row[kRows];
            MmaTile next;
            auto look = [&](int t) {
                if (t >= all) return;
                next = tiles.At(t);
                const int share = kPair ? next.wide / 2 : next.wide;
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const int within = 8 * (part + a.parts * (4 * i + lane / 8)) + lane % 8, r = rank * share + within;
                    row[i] = next.steps > 0 && within < share && r < next.many ? (uint32_t)__ldg(rowOf + next.first + r) : 0;
                }
            };
            look(first);
            for (int t = first; t < all && !failed; t += step) {
                const MmaTile m = next;
                const int share = kPair ? m.wide / 2 : m.wide;
                uint32_t now[kRows];
#pragma unroll
                for (int i = 0; i < kRows; ++i) now[i] = row[i];
                const int eights = (share / 8 - part + a.parts - 1) / a.parts;  // of this part
                look(t + step);
                for (; turn < m.steps; turn += warps) {
                    if (!free()) {
                        failed = true;
                        break;
                    }
                    const uint32_t at = place + ring.stage * a.stageBytes + kMmaABytes + part * 1024;
                    const int col = turn * kMmaDepth + 8 * piece, left = 2 * max(0, min(8, depth - col));  // bytes of the piece
                    const char *const from = x + (left > 0 ? 2ll * col : 0);
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (4 * i + j / 2 >= eights) break;
                            const uint32_t r = __shfl_sync(0xffffffffu, now[i], 4 * j + high);
                            CopyPiece(at + (4 * i + j / 2) * (1024 * a.parts) + (j & 1) * 512 + (j & 1 ? odd : even), from + (uint64_t)r * pitch, left);
                        }
                    }
                    asked();
                }
                turn -= m.steps;
            }
        } else {
            for (int t = first; t < all && !failed; t += step) {
                const MmaTile m = tiles.At(t);
                const int lo = sOffset[m.expert], hi = sOffset[m.expert + 1], f0 = m.f0 + rank * kMmaRows;
                const int share = kPair ? m.wide / 2 : m.wide, c0 = m.first + rank * share, blocks = (share + 63) / 64;
                // the lane's columns of every block: where they are, and how many bytes of its piece exist
                constexpr int kBlocksY = kMmaRows / 64, kBlocksX = kMmaColsMost / (kPair ? 2 : 1) / 64;
                int leftY[kBlocksY], leftX[kBlocksX];
#pragma unroll
                for (int b = 0; b < kBlocksY; ++b) leftY[b] = 2 * max(0, min(8, a.n - f0 - 8 * piece - 64 * b));
#pragma unroll
                for (int b = 0; b < kBlocksX; ++b) leftX[b] = 2 * max(0, min(8, a.d - c0 - 8 * piece - 64 * b));
                const char *const y = static_cast<const char *>(a.dy) + 2ll * (f0 + 8 * piece), *const x = static_cast<const char *>(a.x) + 2ll * (c0 + 8 * piece);
                const uint32_t pitchY = (uint32_t)a.ldy * 2, pitchX = (uint32_t)a.ldx * 2;
                int rowY, rowX;
                auto rows = [&](int k) {  // the part's entry `lane` of a step; -1: none
                    const int at = lo + k * kMmaDepth + 32 * part + lane;
                    rowY = at < hi ? __ldg(a.entries + at) : -1;
                    rowX = at < hi ? (a.byEntry ? rowY : __ldg(a.rows + at)) : -1;
                };
                if (turn < m.steps) rows(turn);
                for (; turn < m.steps; turn += warps) {
                    if (!free()) {
                        failed = true;
                        break;
                    }
                    const uint32_t at = place + ring.stage * a.stageBytes + part * 4096;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t to = at + j * 512 + (j & 1 ? odd : even);
                        const int ry = __shfl_sync(0xffffffffu, rowY, 4 * j + high), rx = __shfl_sync(0xffffffffu, rowX, 4 * j + high);
                        // no row: zeros, from wherever
                        const char *const fromY = y + (uint64_t)(uint32_t)max(ry, 0) * pitchY, *const fromX = x + (uint64_t)(uint32_t)max(rx, 0) * pitchX;
#pragma unroll
                        for (int b = 0; b < kBlocksY; ++b)
                            CopyPiece(to + b * kMmaBlockBytes, leftY[b] > 0 ? fromY + 128 * b : static_cast<const char *>(a.dy), ry < 0 ? 0 : leftY[b]);
#pragma unroll
                        for (int b = 0; b < kBlocksX; ++b) {
                            if (b >= blocks) break;
                            CopyPiece(to + kMmaABytes + b * kMmaBlockBytes, leftX[b] > 0 ? fromX + 128 * b : static_cast<const char *>(a.x), rx < 0 ? 0 : leftX[b]);
                        }
                    }
                    if (turn + warps < m.steps) rows(turn + warps);
                    asked();
                }
                turn -= m.steps;
            }
        }
    } else if (warp == 1 && rank == 0) {
        constexpr bool kAcrossA = kMode != Mode::kProductT, kAcrossB = kMode == Mode::kGrad;
        constexpr uint32_t kType = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
        constexpr uint32_t kInstr = 1u << 4 | kType << 7 | kType << 10 | (uint32_t)kAcrossA << 15 | (uint32_t)kAcrossB << 16 |
                                    (uint32_t)(Tiles<kMode, kPair>::kHigh >> 4) << 24;
        const bool elected = Elected();
        // Of the descriptors only the address changes, and that within 14 bits.
        const uint64_t first64A = OperandAt(base, kAcrossA), first64B = OperandAt(base + kMmaABytes, kAcrossB);
        constexpr int kAlongA = (kAcrossA ? 2048 : 32) >> 4, kAlongB = (kAcrossB ? 2048 : 32) >> 4;
        Ring ring;
        int tile = 0;
        for (int t = first; t < all && !failed; t += step) {
            const MmaTile m = tiles.At(t);
            if (m.steps == 0) continue;
            const int acc = tile & 1, turn = tile >> 1;
            if (turn > 0 && !__all_sync(0xffffffffu, BarWait(sFree + acc, (uint32_t)(turn - 1) & 1u, a.waitCycles))) {
                failed = true;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t shape = kInstr | (uint32_t)(m.wide >> 3) << 17, to = tmem + acc * kMmaColsMost;
            for (int k = 0; k < m.steps; ++k, ring.Next(a.stages)) {
                if (!__all_sync(0xffffffffu, BarWait(sFull + ring.stage, ring.Filled(), a.waitCycles))) {
                    failed = true;
                    break;
                }
                const uint32_t at = (uint32_t)(ring.stage * a.stageBytes) >> 4;
                if (elected) {
#pragma unroll
                    for (int i = 0; i < kMmaDepth / 16; ++i)
                        Mma<kPair>(to, first64A + (at + i * kAlongA), first64B + (at + i * kAlongB), shape, k > 0 || i > 0);
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
    } else if (warp >= 2 && warp < kMmaFirstGather) {
        const int quarter = warp & 3;  // the lanes of tensor memory that the warp may read
        const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
        const int features = kMode == Mode::kProductN ? a.d : a.n;
        Out *const sOut = reinterpret_cast<Out *>(sRaw + (base - Shared(sRaw)) + a.stages * a.stageBytes) + quarter * 1024;
        int tile = 0;
        for (int t = first; t < all; t += step) {
            const MmaTile m = tiles.At(t);
            const int acc = tile & 1, turn = tile >> 1;
            if (m.steps > 0) {
                if (!BarWaitWarp(sDone + acc, (uint32_t)turn & 1u, a.waitCycles + m.steps * kMmaStepCycles)) {
                    failed = true;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                ++tile;
            }
            const int f0 = m.f0 + rank * kMmaRows + quarter * 32;  // the warp's 32 rows of the tile
            int entry = 0;
            const uint32_t from = tmem + ((uint32_t)quarter << 21) + acc * kMmaColsMost;
            if (kMode != Mode::kGrad) entry = lane < m.many ? __ldg(a.entries + m.first + lane) : 0;
            for (int c0 = 0; c0 < m.many; c0 += 32) {
                float v[32] = {};
                if (m.steps > 0) LoadColumns32(from + c0, v);
                if (m.steps > 0 && c0 + 32 >= m.many) {  // all that this warp reads of the accumulator
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) BarArriveAt(LeadersBar(sFree + acc));
                }
                const float by = m.steps > 0 ? alpha : 0.0f;
                const int live = min(32, m.many - c0);
                if constexpr (kMode != Mode::kGrad) {
                    const int now = entry;
                    if (c0 + 32 + lane < m.many) entry = __ldg(a.entries + m.first + c0 + 32 + lane);
                    Out *const out = static_cast<Out *>(a.out);
                    if (a.vectors && beta == 0.0f) {
                        // Through shared memory, so that 16 bytes of a row are stored at once and a row's 32 columns side by side.
                        constexpr int kN = 16 / (int)sizeof(Out), kPieces = 32 / kN;
#pragma unroll
                        for (int i = 0; i < 32; ++i) sOut[32 * i + lane] = FromFloat<Out>(by * v[i]);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            const int c = (32 * i + lane) / kPieces, at = lane % kPieces * kN;
                            const long long row = __shfl_sync(0xffffffffu, now, c);
                            const uint4 piece = *reinterpret_cast<const uint4 *>(sOut + 32 * c + at);
                            Out *const to = out + row * a.ldo + f0 + at;
                            if (c < live && f0 + at + kN <= features) *reinterpret_cast<uint4 *>(to) = piece;
                            else if (c < live)  // the last columns
                                for (int j = 0; f0 + at + j < features; ++j) to[j] = sOut[32 * c + at + j];
                        }
                        __syncwarp();
                    } else {
                        // A column a lane.  What is read is asked for before anything is stored.
                        const bool in = f0 + lane < features;
#pragma unroll
                        for (int g = 0; g < 32; g += 8) {
                            float old[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const long long row = __shfl_sync(0xffffffffu, now, g + i);
                                old[i] = beta != 0.0f && in && g + i < live ? ToFloat(out[row * a.ldo + f0 + lane]) : 0.0f;
                            }
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const long long row = __shfl_sync(0xffffffffu, now, g + i);
                                const float u = beta != 0.0f ? fmaf(beta, old[i], by * v[g + i]) : by * v[g + i];
                                if (in && g + i < live) out[row * a.ldo + f0 + lane] = FromFloat<Out>(u);
                            }
                        }
                    }
                } else {
                    constexpr int kN = 16 / (int)sizeof(Out), kPieces = 32 / kN;
                    Out *const out = static_cast<Out *>(a.out) + ((long long)m.expert * a.n + f0) * a.ldo + m.first + c0;
                    if (beta == 0.0f) {
                        // The lane's row, its pieces exchanged so that neither side meets in a bank; then pieces of a row side by side, or where
                        // rows do not start on 16 bytes a row at a time.
                        auto pieceOf = [&](int r, int at) { return sOut + 32 * r + kN * (at ^ (r * kPieces / 8 & (kPieces - 1))); };
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            float u[kN];
#pragma unroll
                            for (int j = 0; j < kN; ++j) u[j] = by * v[kN * i + j];
                            StoreFloats<Out, kN, true>(pieceOf(lane, i), u);
                        }
                        __syncwarp();
                        if (a.vectors) {
#pragma unroll
                            for (int i = 0; i < kPieces; ++i) {
                                const int r = (32 * i + lane) / kPieces, at = lane % kPieces;
                                const uint4 piece = *reinterpret_cast<const uint4 *>(pieceOf(r, at));
                                Out *const to = out + r * a.ldo + kN * at;
                                if (f0 + r < features && kN * (at + 1) <= live) *reinterpret_cast<uint4 *>(to) = piece;
                                else if (f0 + r < features)  // the last columns
                                    for (int j = 0; kN * at + j < live; ++j) to[j] = pieceOf(r, at)[j];
                            }
                        } else {
#pragma unroll 8
                            for (int r = 0; r < 32; ++r) {
                                const Out one = pieceOf(r, lane / kN)[lane % kN];
                                if (f0 + r < features && lane < live) out[r * a.ldo + lane] = one;
                            }
                        }
                        __syncwarp();
                    } else if (f0 + lane < features) {
                        // A row a lane, each access 32 sectors: 8192 entries of 16 experts, 1024 x 2048, 941 us into f32 and 2030 into 16 bits,
                        // where beta = 0 takes 67 and 55.
                        Out *const to = out + lane * a.ldo;
#pragma unroll
                        for (int g = 0; g < 32; g += 8) {
                            float old[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) old[i] = g + i < live ? ToFloat(to[g + i]) : 0.0f;
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (g + i < live) to[g + i] = FromFloat<Out>(fmaf(beta, old[i], by * v[g + i]));
                        }
                    }
                }
            }
        }
    }
    __syncwarp();
    if (failed) atomicMax(&gExpertsError, kWaitRanOut);
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

// Of stacked matrices, `high` rows of 64 elements of one, swizzled.
inline bool MapOf(CUtensorMap *map, aclDataType type, const void *at, long long cols, long long rows, long long ld, int deep, int high)
{
    const EncodeTiled encode = Encoder();
    if (encode == nullptr) return false;
    const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)deep};
    const cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(ld * 2 * rows)};
    const cuuint32_t box[3] = {64, (cuuint32_t)high, 1}, step[3] = {1, 1, 1};
    return encode(map, type == ACL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void *>(at), size, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Entries of a tile: as many as an expert has on average, half as much again for the uneven ones, so that the weights of most experts are
// read by one tile a column block, and stages are no larger than that wants.  32 experts of 2048 x 2048, four a token, us with tiles of 256, 128
// (pairs of CTAs) and 64 entries: 64 tokens 54, 53, 54; 512 tokens 64, 62, 81; 1024 tokens 69, 79, 117; 4096 tokens 135, 182, 353.
inline int TileColumns(long long nnz, long long experts)
{
    const long long want = (nnz * 3 + 2 * experts - 1) / (2 * experts);
    int cols = 32;
    while (cols < kMmaColsMost && cols < want) cols *= 2;
    return cols;
}

long long gExpertsWaitCycles = kMmaWaitCycles;
unsigned gExpertsExtraTx = 0;

template <typename T, typename Out, Mode kMode, bool kPair>
cudaError_t LaunchTiles(MmaArgs a, const CUtensorMap &mapW, cudaStream_t stream)
{
    a.stageBytes = kMmaABytes + a.colsMost * 128 / (kPair ? 2 : 1);
    a.stages = std::min(kMmaShared / a.stageBytes, kMmaStagesMost);
    // Few rows are one warp's, so that more stages are on their way: with two warps at each of six stages a step of a tile of 32 entries takes 300 ns.
    a.parts = kMode != Mode::kGrad && a.colsMost <= kMmaColsMost / kMmaPartsMost / (kPair ? 2 : 1) ? 1 : kMmaPartsMost;
    a.waitCycles = gExpertsWaitCycles;
    a.extraTx = gExpertsExtraTx;
    const auto kernel = ExpertsTensorKernel<T, Out, kMode, kPair>;
    const cudaError_t e = AllowShared<ExpertsTensorKernel<T, Out, kMode, kPair>>(kMmaShared + kMmaStoreBytes<Out> + 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(b200sp_sm_count() / 2 * 2));
    cfg.blockDim = dim3(kMmaThreads);
    cfg.dynamicSmemBytes = (size_t)(a.stages * a.stageBytes + kMmaStoreBytes<Out> + 1024);
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
    return cudaLaunchKernelEx(&cfg, kernel, a, mapW);
}

// A pair of CTAs on a tile of 256 columns reads half as much of X (or of both operands of a gradient) per product.  That counts where there are
// products enough to be bound by them: 1024 tokens as above 69 us, by single CTAs 84, 4096 tokens 135 and 178; gradients of 4096 entries of 1024 x
// 2048 87 and 102.  With few entries there is nothing in it (64 tokens 54 and 54).
template <typename T, typename Out, Mode kMode>
cudaError_t LaunchTensor(const MmaArgs &a, const CUtensorMap &mapW, cudaStream_t stream)
{
    const int features = kMode == Mode::kProductN ? a.d : a.n;
    return a.colsMost >= 128 && features > kMmaRows ? LaunchTiles<T, Out, kMode, true>(a, mapW, stream)
                                                    : LaunchTiles<T, Out, kMode, false>(a, mapW, stream);
}
