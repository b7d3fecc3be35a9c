// Stable sort of small integer keys by one thread-block cluster, one launch.
//
// Radix sort from the lowest digit. The cluster's warps own consecutive stretches of the input. A
// pass counts each warp's digits in shared memory, adds the counts up over warps, blocks (through
// distributed shared memory) and digits, and then every warp walks its stretch in order again and
// writes each element to its place: equal digits keep their order, whatever the timing. Elements
// between passes travel through global memory (L2); the barrier between passes is the hardware's
// cluster barrier, so there is nothing to spin on. Bound by latency: at 65536 keys a warp has 8
// steps of 32 keys in each of two walks per pass.
#pragma once

#include "kernels/ops_common.cuh"

#include <cooperative_groups.h>

namespace bccl {
namespace ops {

constexpr int kSortMaxBits = 10;  // digit width: 1024 bins x 32 warps of counters fill 128 KiB

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

// One pass over n elements by digit (key >> shift) & (2^bits - 1). get(i) gives {key, position};
// put(place, key, position) stores it; totals(digit, first place) is called once per digit by block 0.
// counters: [warps][2^bits] and then 2 x 2^bits words of shared memory.
template <typename Get, typename Put, typename Totals>
__device__ __forceinline__ void sort_pass(unsigned int* counters, long long n, int shift, int bits, Get get, Put put,
                                          Totals totals) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int nbins = 1 << bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int rank = static_cast<int>(cluster.block_rank()), blocks = static_cast<int>(cluster.num_blocks());
    unsigned int* mine = counters + warp * nbins;
    unsigned int* block_total = counters + warps * nbins;  // read by the other blocks
    unsigned int* place = block_total + nbins;             // scratch of the scan over digits
    const long long per = ((n + static_cast<long long>(warps) * blocks * 32 - 1) / (static_cast<long long>(warps) * blocks * 32)) * 32;
    const long long lo = min(n, (static_cast<long long>(rank) * warps + warp) * per), hi = min(n, lo + per);
    const unsigned int mask = nbins - 1;

    for (int i = threadIdx.x; i < warps * nbins; i += blockDim.x) counters[i] = 0;
    __syncthreads();
    for (long long i = lo + lane; i < hi + lane; i += 32) {  // the same trips for every lane
        const bool in = i < hi;
        const unsigned int d = in ? (get(i).x >> shift) & mask : nbins;
        const unsigned int same = __match_any_sync(0xffffffffu, d);
        if (in && lane == __ffs(same) - 1) mine[d] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // Counts of the warps before this one, and the block's total, per digit.
    for (int d = threadIdx.x; d < nbins; d += blockDim.x) {
        unsigned int sum = 0;
        for (int w = 0; w < warps; ++w) {
            const unsigned int c = counters[w * nbins + d];
            counters[w * nbins + d] = sum;
            sum += c;
        }
        block_total[d] = sum;
    }
    cluster.sync();
    for (int d = threadIdx.x; d < nbins; d += blockDim.x) {
        unsigned int before = 0, all = 0;
        for (int b = 0; b < blocks; ++b) {
            const unsigned int c = cluster.map_shared_rank(block_total, b)[d];
            if (b < rank) before += c;
            all += c;
        }
        place[d] = all;
        for (int w = 0; w < warps; ++w) counters[w * nbins + d] += before;
    }
    __syncthreads();
    // Exclusive sum over digits, by one warp.
    if (warp == 0) {
        unsigned int run = 0;
        for (int d0 = 0; d0 < nbins; d0 += 32) {
            const int d = d0 + lane;
            const unsigned int v = d < nbins ? place[d] : 0;
            unsigned int incl = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned int t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            if (d < nbins) place[d] = run + incl - v;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    __syncthreads();
    if (rank == 0)
        for (int d = threadIdx.x; d < nbins; d += blockDim.x) totals(static_cast<unsigned int>(d), place[d]);
    for (long long i = lo + lane; i < hi + lane; i += 32) {
        const bool in = i < hi;
        const uint2 kp = in ? get(i) : make_uint2(0, 0);
        const unsigned int d = in ? (kp.x >> shift) & mask : nbins;
        const unsigned int same = __match_any_sync(0xffffffffu, d);
        const int leader = __ffs(same) - 1;
        unsigned int base = 0;
        if (in && lane == leader) {
            base = mine[d];
            mine[d] = base + __popc(same);
        }
        base = __shfl_sync(0xffffffffu, base, leader);
        if (in) put(place[d] + base + __popc(same & ((1u << lane) - 1)), kp.x, kp.y);
        __syncwarp();
    }
    // The next pass reads what all blocks wrote; and no block may leave, or reuse its totals,
    // while another reads them.
    cluster.sync();
}

// Blocks of the cluster and their size for n elements: one block while it has few steps per warp.
inline int sort_blocks(long long n) { return n <= 4096 ? 1 : 8; }
inline size_t sort_smem(int threads, int bits) {
    return sizeof(unsigned int) * (static_cast<size_t>(threads / 32) + 2) * (1u << bits);
}

}  // namespace ops
}  // namespace bccl
