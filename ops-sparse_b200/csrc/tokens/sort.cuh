// Positions in the order of their keys, stable: a radix sort by one thread-block cluster, in one launch.
//
// The token operators sort few and small things -- thousands of positions by token, or by expert -- in the middle of a chain of
// kernels, where launches cost more than the sort.  So every pass over a digit (up to ten bits: one pass for experts, two for
// the tokens of a large table) is one phase of a kernel of up to eight CTAs, each with a contiguous share of the positions:
// count the digits of the share in shared memory; read the other CTAs' counts through the cluster, which gives every digit's
// first place; then rank tile by tile (by warp, step and lane, which is the order in memory) and store.  Passes meet at
// cluster barriers.  Nothing is atomic across CTAs, so the result is unique and the same in every run.
// One B200: 128 entries by 64 experts 5 us, 32,768 some 13, 131,072 40 and 1,048,576 285 (one pass; from 32,768 on time grows with the count, since
// the cluster is as large as it gets); 16,384 tokens of a table of 65,536 rows (two passes) less than 20,
// with 64 MB of zeros written beside them.  What bounds it is latency: loads, barriers and the cluster's reads one after the other.
#pragma once

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "tokens/common.cuh"

namespace b200sp_tokens {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortSteps = 4;                            // positions per thread and tile
constexpr int kSortTile = kSortThreads * kSortSteps;
constexpr int kSortMaxBits = 10;
constexpr int kSortMaxCtas = 8;                          // the portable cluster size

struct SortArgs {
    const void *keys;     // int32 or int64, the caller's
    int count, limit;     // keys outside [0, limit) count as limit
    int passes, digitBits;
    int *keyA, *posA;     // sorted, after the last pass
    int *keyB, *posB;     // between passes (unused with one pass)
    int *offsets;         // with one pass, or nullptr: first place of every key 0 ... limit, and the end, limit + 2 numbers
};

inline int SortBits(long long limit)  // of the numbers 0 ... limit
{
    int bits = 1;
    while ((1ll << bits) <= limit) ++bits;
    return bits;
}
inline void SortPasses(long long limit, long long count, SortArgs *a)
{
    // in several passes a tile of its own lies beside the counts of a digit
    const int bits = SortBits(limit), most = bits > kSortMaxBits && count <= kSortTile ? kSortMaxBits - 1 : kSortMaxBits;
    a->passes = (bits + most - 1) / most;
    a->digitBits = (bits + a->passes - 1) / a->passes;
}
// Up to a tile one CTA, which keeps the positions in shared memory between the passes.
inline int SortCtas(long long count)
{
    int ctas = 1;
    while (ctas < kSortMaxCtas && count > kSortTile && count > (long long)ctas * kSortTile / 2) ctas *= 2;
    return ctas;
}
// Shared memory: a word and a count per warp and digit, three numbers per digit; a tile's keys and positions.
inline int SortShared(int digitBits, bool tile) { return (1 << digitBits) * (kSortWarps * 6 + 3 * 4) + (tile ? kSortTile * 8 : 0); }
constexpr int kSortSharedMost = (1 << kSortMaxBits) * (kSortWarps * 6 + 3 * 4);
static_assert((1 << (kSortMaxBits - 1)) * (kSortWarps * 6 + 3 * 4) + kSortTile * 8 <= kSortSharedMost);

template <typename Key> __device__ __forceinline__ int SortKey(const SortArgs &a, int i)
{
    const Key k = static_cast<const Key *>(a.keys)[i];
    return k < 0 || k >= (Key)a.limit ? a.limit : (int)k;
}

// Rank of the lane's position among its warp's of the same digit so far: the lanes of a digit find each other through its word
// (mask: zero before and after).
__device__ __forceinline__ int RankInWarp(uint32_t *mask, uint16_t *count, int d, bool in, int lane)
{
    if (in) atomicOr(mask + d, 1u << lane);
    __syncwarp();
    uint32_t peers = 0;
    int had = 0;
    if (in) {
        peers = *static_cast<volatile uint32_t *>(mask + d);
        had = *static_cast<volatile uint16_t *>(count + d);
    }
    const int among = __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (in && among == 0) {
        mask[d] = 0;
        count[d] = (uint16_t)(had + __popc(peers));
    }
    __syncwarp();
    return had + among;
}
// A digit's counts by warp become the places of every warp's first; returns their sum.
__device__ __forceinline__ int PlacesByWarp(uint16_t *counts, int bins, int warps)
{
    int run = 0;
    for (int w = 0; w < warps; w += 8) {
        int n[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) n[u] = w + u < warps ? counts[(w + u) * bins] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (w + u < warps) counts[(w + u) * bins] = (uint16_t)run;
            run += n[u];
        }
    }
    return run;
}
// Inclusive sums over the CTA's threads.
__device__ __forceinline__ int SumsBefore(int own, int *sScan)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += t;
    }
    if (lane == 31) sScan[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int w = sScan[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, w, d);
            if (lane >= d) w += t;
        }
        sScan[lane] = w;
    }
    __syncthreads();
    return incl + (warp > 0 ? sScan[warp - 1] : 0);
}

// At most a tile, by one CTA: a thread holds four positions, which change places through shared memory.
template <typename Key, typename Place> __device__ __forceinline__ void TileSort(const SortArgs &a, unsigned char *shared, Place &&place)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << a.digitBits;
    uint32_t *const sMask = reinterpret_cast<uint32_t *>(shared);            // [warp][digit]
    int *const sBase = reinterpret_cast<int *>(sMask + kSortWarps * bins);   // [digit]
    uint16_t *const sWarp = reinterpret_cast<uint16_t *>(sBase + 3 * bins);  // [warp][digit]
    int2 *const sTile = reinterpret_cast<int2 *>(sWarp + kSortWarps * bins);
    __shared__ int sScan[kSortWarps];
    // As few warps as have positions, 128 each; the others only help to count.
    const int warps = (a.count + 32 * kSortSteps - 1) / (32 * kSortSteps), first = warp * (32 * kSortSteps) + lane;
    int key[kSortSteps], pos[kSortSteps];
#pragma unroll
    for (int u = 0; u < kSortSteps; ++u) {
        pos[u] = first + 32 * u;
        key[u] = pos[u] < a.count ? SortKey<Key>(a, pos[u]) : -1;
    }
    for (int i = tid; i < warps * bins; i += kSortThreads) sMask[i] = 0;
    for (int p = 0; p < a.passes; ++p) {
        const bool last = p == a.passes - 1;
        const int shift = p * a.digitBits;
        for (int i = tid; i < warps * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t *>(sWarp)[i] = 0;
        __syncthreads();
        int at[kSortSteps];
        if (warp < warps) {
#pragma unroll
            for (int u = 0; u < kSortSteps; ++u)
                at[u] = RankInWarp(sMask + warp * bins, sWarp + warp * bins, (key[u] >> shift) & (bins - 1), key[u] >= 0, lane);
        }
        __syncthreads();
        const int own = tid < bins ? PlacesByWarp(sWarp + tid, bins, warps) : 0;
        const int start = SumsBefore(own, sScan) - own;
        if (tid < bins) {
            sBase[tid] = start;
            if (a.offsets != nullptr && tid <= a.limit + 1) a.offsets[tid] = start;
            // 2^bits > limit: the end of the last key has a digit of its own unless the digits are used up
            if (a.offsets != nullptr && tid == a.limit && a.limit + 1 == bins) a.offsets[bins] = a.count;
        }
        __syncthreads();
        if (warp < warps) {
#pragma unroll
            for (int u = 0; u < kSortSteps; ++u) {
                if (key[u] < 0) continue;
                const int d = (key[u] >> shift) & (bins - 1), to = sBase[d] + sWarp[warp * bins + d] + at[u];
                if (!last) {
                    sTile[to] = make_int2(key[u], pos[u]);
                } else {
                    a.keyA[to] = key[u];
                    a.posA[to] = pos[u];
                    place(key[u], pos[u], to);
                }
            }
        }
        __syncthreads();  // the caller may read what was stored
        if (last) break;
#pragma unroll
        for (int u = 0; u < kSortSteps; ++u) {
            if (first + 32 * u >= a.count) continue;
            key[u] = sTile[first + 32 * u].x;
            pos[u] = sTile[first + 32 * u].y;
        }
    }
}

// All CTAs of the cluster, 1024 threads each; place(key, position, where) is told of every position in the last pass.
template <typename Key, typename Place> __device__ __forceinline__ void ClusterSort(const SortArgs &a, unsigned char *shared, Place &&place)
{
    if (a.count <= kSortTile) {
        TileSort<Key>(a, shared, place);
        return;
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int bins = 1 << a.digitBits;
    uint32_t *const sMask = reinterpret_cast<uint32_t *>(shared);          // [warp][digit]
    int *const sCount = reinterpret_cast<int *>(sMask + kSortWarps * bins);  // [digit]: this CTA's
    int *const sBase = sCount + bins;                                      // [digit]: next place
    int *const sTile = sBase + bins;                                       // [digit]: of the tile (the others may still read sCount)
    uint16_t *const sWarp = reinterpret_cast<uint16_t *>(sTile + bins);    // [warp][digit]
    __shared__ int sScan[kSortWarps];
    // shares of whole warps' segments
    const int share = ((a.count + ctas - 1) / ctas + 31) / 32 * 32;
    const int lo = min((long long)a.count, (long long)rank * share), hi = min((long long)a.count, (long long)lo + share);
    for (int i = tid; i < kSortWarps * bins; i += kSortThreads) sMask[i] = 0;
    for (int p = 0; p < a.passes; ++p) {
        const bool last = p == a.passes - 1;
        const int shift = p * a.digitBits;
        // the last pass ends in A
        const bool fromA = (a.passes - p) % 2 == 0;
        const int *const keyIn = fromA ? a.keyA : a.keyB, *const posIn = fromA ? a.posA : a.posB;
        int *const keyOut = fromA ? a.keyB : a.keyA, *const posOut = fromA ? a.posB : a.posA;
        int key[kSortSteps], pos[kSortSteps], at[kSortSteps];
        // The tile's positions, and their ranks among the warps' of the same digit; then sTile has the tile's counts.
        auto rankTile = [&](int tile) {
            for (int i = tid; i < kSortWarps * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t *>(sWarp)[i] = 0;
            const int first = tile + warp * (32 * kSortSteps) + lane;
#pragma unroll
            for (int u = 0; u < kSortSteps; ++u) {
                const int i = first + 32 * u;
                key[u] = -1;
                if (i < hi) {
                    key[u] = p == 0 ? SortKey<Key>(a, i) : __ldcg(keyIn + i);
                    pos[u] = p == 0 ? i : __ldcg(posIn + i);
                }
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kSortSteps; ++u)
                at[u] = RankInWarp(sMask + warp * bins, sWarp + warp * bins, (key[u] >> shift) & (bins - 1), key[u] >= 0, lane);
            __syncthreads();
            if (tid < bins) sTile[tid] = PlacesByWarp(sWarp + tid, bins, kSortWarps);
        };
        // A share of one tile is read once; of a longer one the digits are counted first.
        const bool once = hi - lo <= kSortTile;
        if (once) {
            rankTile(lo);
            if (tid < bins) sCount[tid] = sTile[tid];
        } else {
            for (int i = tid; i < bins; i += kSortThreads) sCount[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += kSortThreads) {
                const int k = p == 0 ? SortKey<Key>(a, i) : __ldcg(keyIn + i);
                atomicAdd(sCount + ((k >> shift) & (bins - 1)), 1);
            }
        }
        cluster.sync();
        int all = 0, before = 0;  // of digit tid
        if (tid < bins) {
            int n[kSortMaxCtas];
#pragma unroll
            for (int c = 0; c < kSortMaxCtas; ++c) n[c] = c < ctas ? cluster.map_shared_rank(sCount, c)[tid] : 0;
#pragma unroll
            for (int c = 0; c < kSortMaxCtas; ++c) {
                before += c < rank ? n[c] : 0;
                all += n[c];
            }
        }
        const int start = SumsBefore(all, sScan) - all;
        if (tid < bins) {
            sBase[tid] = start + before;
            if (a.offsets != nullptr && rank == 0 && tid <= a.limit + 1) a.offsets[tid] = start;
            // 2^bits > limit: the end of the last key has a digit of its own unless the digits are used up
            if (a.offsets != nullptr && rank == 0 && tid == a.limit && a.limit + 1 == bins) a.offsets[bins] = a.count;
        }
        for (int tile = lo; tile < hi; tile += kSortTile) {
            if (!once) rankTile(tile);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kSortSteps; ++u) {
                if (key[u] < 0) continue;
                const int d = (key[u] >> shift) & (bins - 1);
                const int to = sBase[d] + sWarp[warp * bins + d] + at[u];
                keyOut[to] = key[u];
                posOut[to] = pos[u];
                if (last) place(key[u], pos[u], to);
            }
            __syncthreads();
            if (tid < bins) sBase[tid] += sTile[tid];
        }
        cluster.sync();  // what was stored is read by the others from here on
    }
}

}  // namespace b200sp_tokens
