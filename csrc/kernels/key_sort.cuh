// Stable sort of small integer keys.
//
// Radix sort from the lowest digit. Warps own consecutive stretches of the input. A pass counts each
// warp's digits in shared memory, adds the counts up over warps, blocks and digits, and then every
// warp walks its stretch in order again and writes each element to its place: equal digits keep their
// order, whatever the timing. Elements between passes travel through global memory (L2).
//
// Up to 32768 elements one thread-block cluster does all passes in one launch: blocks read each other's
// totals through distributed shared memory, and the barrier between passes is the hardware's cluster
// barrier, so there is nothing to spin on. More elements get two launches per pass over up to 128 blocks
// (count, then place), with the totals in global memory: 800000 keys of 4 bits take 28 us that way and 144 us
// on a cluster.
//
// Bound by latency: a warp loads kBatch steps of 32 keys at once, and stretches of one batch stay in
// registers for the second walk. Lanes with equal digits are found by a vote per bit, all in flight
// together (65536 keys of 7 bits on a cluster: 23 us with match.any, 19 with votes in a loop, 16 unrolled);
// the votes are two thirds of the counting.
#pragma once

#include "kernels/ops_common.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace bccl {
namespace ops {

constexpr int kSortWarps = 32;
constexpr int kSortMaxBits = 10;  // digit width: 1024 bins, a thread each; x 32 warps of counters fill 128 KiB
constexpr int kBatch = 8;

// Key of element i: ids[i] - first where that lies in [0, bins), else `bins` (sorted last).
struct KeySource {
    const void* ids;
    int ids64;
    long long first, bins, skip;
    int has_skip;
    __device__ __forceinline__ unsigned int operator()(long long i) const {
        const long long id = ids64 ? __ldg(static_cast<const long long*>(ids) + i)
                                   : static_cast<long long>(__ldg(static_cast<const int*>(ids) + i));
        // Compared before subtracting: any 64-bit id is safe.
        const bool in = id >= first && id - first < bins && !(has_skip && id == skip);
        return static_cast<unsigned int>(in ? id - first : bins);
    }
};

// The lanes of `valid` whose BITS-bit digit equals this lane's (which must be one of them).
template <int BITS>
__device__ __forceinline__ unsigned int same_digit(unsigned int d, unsigned int valid) {
    unsigned int votes[BITS];
#pragma unroll
    for (int b = 0; b < BITS; ++b) votes[b] = __ballot_sync(0xffffffffu, (d >> b) & 1);
#pragma unroll
    for (int b = 0; b < BITS; ++b) valid &= (d >> b) & 1 ? votes[b] : ~votes[b];
    return valid;
}

// How the blocks of a pass learn of each other's totals. kCount ends a pass after writing them to
// global memory, kPlace takes them from there.
enum SortMode { kCluster, kCount, kPlace };

__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// One pass over n elements by digit (key >> shift) & (2^BITS - 1), blockDim.x == 1024. get(i) gives
// {key, position}; put(place, key, position) stores it; totals(digit, first place) is called once
// per digit by block 0. counters: shared memory of sort_smem(BITS) bytes. grid_totals ([blocks][2^BITS], not
// for kCluster). After the last pass other blocks' elements may still be on their way.
template <int BITS, SortMode MODE, typename Get, typename Put, typename Totals>
__device__ __forceinline__ void sort_pass(unsigned int* counters, unsigned int* grid_totals, long long n, int shift,
                                          bool last, Get get, Put put, Totals totals) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int kBins = 1 << BITS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = MODE == kCluster ? static_cast<int>(cluster.block_rank()) : static_cast<int>(blockIdx.x);
    const int blocks = MODE == kCluster ? static_cast<int>(cluster.num_blocks()) : static_cast<int>(gridDim.x);
    const unsigned int lower = (1u << lane) - 1;
    unsigned int* mine = counters + warp * kBins;
    unsigned int* block_total = counters + kSortWarps * kBins;  // read by the other blocks
    unsigned int* start = block_total + kBins;                  // where this block's elements of a digit go
    unsigned int* warp_total = start + kBins;
    const long long share = static_cast<long long>(kSortWarps) * blocks * 32;
    const long long per = (n + share - 1) / share * 32;
    const long long lo = min(n, (static_cast<long long>(rank) * kSortWarps + warp) * per), hi = min(n, lo + per);

    uint2 held[kBatch];
    unsigned int equal[kBatch];
    auto load = [&](long long i0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const long long i = i0 + b * 32 + lane;
            held[b] = i < hi ? get(i) : make_uint2(0, 0);
        }
    };
    load(lo);
    for (int i = threadIdx.x; i < kSortWarps * kBins / 4; i += blockDim.x)
        reinterpret_cast<uint4*>(counters)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (long long i0 = lo; i0 < hi; i0 += kBatch * 32) {
        if (i0 != lo) load(i0);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i0 + b * 32 >= hi) break;
            const bool in = i0 + b * 32 + lane < hi;
            const unsigned int d = (held[b].x >> shift) & (kBins - 1);
            equal[b] = same_digit<BITS>(d, __ballot_sync(0xffffffffu, in));
            if (in && (equal[b] & lower) == 0) mine[d] += __popc(equal[b]);
            __syncwarp();
        }
    }
    __syncthreads();
    // A thread per digit: counts of the warps before each warp, the block's total, the blocks' totals.
    const int d = threadIdx.x;
    unsigned int before = 0, all = 0;
    if (d < kBins) {
        unsigned int c[kSortWarps];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) c[w] = counters[w * kBins + d];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            counters[w * kBins + d] = all;
            all += c[w];
        }
        block_total[d] = all;
        if constexpr (MODE == kCount) grid_totals[rank * kBins + d] = all;
    }
    if constexpr (MODE == kCount) return;
    if constexpr (MODE == kPlace) {
        all = 0;
        if (d < kBins) {
#pragma unroll 16
            for (int b = 0; b < blocks; ++b) {
                const unsigned int c = __ldg(grid_totals + b * kBins + d);
                if (b < rank) before += c;
                all += c;
            }
        }
    } else if (blocks > 1) {
        cluster.sync();
        all = 0;
        if (d < kBins) {
#pragma unroll 8
            for (int b = 0; b < blocks; ++b) {
                const unsigned int c = cluster.map_shared_rank(block_total, b)[d];
                if (b < rank) before += c;
                all += c;
            }
        }
        cluster_arrive_relaxed();  // done with the other blocks' totals
    }
    // Exclusive sum over the digits.
    unsigned int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    if (lane == 31) warp_total[warp] = incl;
    __syncthreads();
    unsigned int first = lane < warp ? warp_total[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(0xffffffffu, first, o);
    first += incl - all;
    if (d < kBins) {
        if (rank == 0) totals(static_cast<unsigned int>(d), first);
        start[d] = first + before;
    }
    __syncthreads();
    for (long long i0 = lo; i0 < hi; i0 += kBatch * 32) {
        const bool again = per > kBatch * 32;
        if (again) load(i0);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i0 + b * 32 >= hi) break;
            const bool in = i0 + b * 32 + lane < hi;
            const unsigned int dg = (held[b].x >> shift) & (kBins - 1);
            if (again) equal[b] = same_digit<BITS>(dg, __ballot_sync(0xffffffffu, in));
            const unsigned int at = mine[dg];
            __syncwarp();
            if (in && (equal[b] & lower) == 0) mine[dg] = at + __popc(equal[b]);
            __syncwarp();
            if (in) put(start[dg] + at + __popc(equal[b] & lower), held[b].x, held[b].y);
        }
    }
    if (MODE == kPlace) return;
    if (blocks > 1) {
        cluster_wait();             // nobody reads this block's totals any more
        if (!last) cluster.sync();  // the next pass reads what all blocks wrote
    } else if (!last) {
        __syncthreads();
    }
}

inline size_t sort_smem(int bits) {
    return sizeof(unsigned int) * (static_cast<size_t>(kSortWarps + 2) * (1u << bits) + kSortWarps);
}

// Digit widths that kernels exist for (votes are unrolled), and the one to use for `bits`.
template <typename F>
cudaError_t with_bits(int bits, F&& f) {
    if (bits <= 4) return f(Int<4>{});
    if (bits <= 7) return f(Int<7>{});
    if (bits <= 9) return f(Int<9>{});
    return f(Int<10>{});
}

// Elements that a cluster sorts in one launch. By cluster and by grid, us: sorts of 4, 7 and 9 bits of 32768 keys
// 7.8, 9.5, 11.1 and 10.2, 11.0, 12.2; of 65536 11.2, 14.7, 16.9 and 11.5, 12.0, 13.0; a gradient whose keys
// take two passes (rows of 16 bytes, 128256 of them) 36 and 40 with 32768 positions, 51 and 46 with 65536.
constexpr long long kClusterSort = 32768;

// Blocks of the launches for more elements: 2048 each while that is no more than 128.
inline int sort_grid(long long n) { return static_cast<int>(std::min(128ll, ceil_div(n, 2048))); }
// Words of grid_totals that sorting n elements needs.
inline size_t sort_totals(long long n) {
    return n <= kClusterSort ? 0 : static_cast<size_t>(sort_grid(n)) << kSortMaxBits;
}

// Launches a kernel of sort passes: by a cluster (one block while a warp has at most two steps, else 8,
// the most that every GPU guarantees), or by the blocks of sort_grid.
template <typename... Params, typename... Args>
cudaError_t launch_sort(void (*kernel)(Params...), bool by_cluster, long long n, int bits, cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = !by_cluster || n <= kSortWarps * 2 * 32 ? 1 : 8;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(by_cluster ? attr[0].val.clusterDim.x : sort_grid(n));
    cfg.blockDim = dim3(kSortWarps * 32);
    cfg.dynamicSmemBytes = sort_smem(bits);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cfg.dynamicSmemBytes > 48 * 1024) {  // more than a kernel may have unasked
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(sort_smem(kSortMaxBits)));
        if (e != cudaSuccess) return e;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace ops
}  // namespace bccl
