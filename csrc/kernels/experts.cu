// Tokens sorted by expert and back, with weights applied, and the gradients.
//
// Assignment a = t * top + j sends token t to expert ids[a]; slots[a] is its row after sorting.
//   dispatch          rows[slots[a]] = x[t]                    reads T rows, writes T * top
//   combine           y[t] = sum_j w[a] * rows[slots[a]]       reads T * top rows, writes T
//   combine backward  drows[slots[a]] = w[a] * dy[t], dw[a] = <dy[t], rows[slots[a]]>
//   dispatch backward = combine without weights
//
// Everything is done by token: a block holds its token's row in registers and visits the rows of
// its assignments, so a token's row is read (or written) once and no two blocks write one row.
// Bound by memory.
#include "kernels/key_sort.cuh"
#include "kernels/ops.h"

#include <algorithm>

namespace bccl {
namespace ops {
namespace {

// One pass: the digits are the experts themselves and `experts` for dropped assignments.
template <int BITS, SortMode MODE>
__global__ void __launch_bounds__(1024) expert_sort_kernel(const KeySource key, long long n, unsigned int* grid_totals,
                                                           int* slots, int* sources, int* offsets) {
    extern __shared__ unsigned int counters[];
    const unsigned int experts = static_cast<unsigned int>(key.bins);
    sort_pass<BITS, MODE>(
        counters, grid_totals, n, 0, true, [&](long long i) { return make_uint2(key(i), static_cast<unsigned int>(i)); },
        [&](unsigned int place, unsigned int k, unsigned int a) {
            slots[a] = k < experts ? static_cast<int>(place) : -1;
            sources[place] = k < experts ? static_cast<int>(a) : -1;
        },
        [&](unsigned int d, unsigned int first) {
            if (d <= experts) offsets[d] = static_cast<int>(first);
        });
}

constexpr int kTokenThreads = 256;

// Dropped assignments have slot -1; nothing outside the rows is touched whatever the slots hold.
__device__ __forceinline__ bool in_rows(int slot, long long n) { return static_cast<unsigned int>(slot) < n; }

// blockIdx.x walks tokens and then, past them, the rows behind the last kept one; blockIdx.y columns.
template <int D, int E>
__global__ void __launch_bounds__(kTokenThreads) dispatch_kernel(const Bits<D>* __restrict__ x, long long x_stride,
                                                                 const int* __restrict__ slots,
                                                                 const int* __restrict__ kept, long long tokens, int top,
                                                                 long long h, Bits<D>* __restrict__ rows) {
    const long long c = (static_cast<long long>(blockIdx.y) * blockDim.x + threadIdx.x) * E;
    if (c >= h) return;
    for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
        const Raw<D, E> r = load_raw_cs<D, E>(x + t * x_stride + c);
        const int* s = slots + t * top;
        for (int j = 0; j < top; ++j) {
            const int slot = __ldg(s + j);
            if (in_rows(slot, tokens * top)) store_raw_cs<D, E>(rows + static_cast<long long>(slot) * h + c, r);
        }
    }
    for (long long i = __ldg(kept) + static_cast<long long>(blockIdx.x); i < tokens * top; i += gridDim.x)
        store_raw_cs<D, E>(rows + i * h + c, zero_raw<D, E>());
}

// U rows are in flight per thread; each token's sum runs over j in order.
template <int D, int WD, int E, int U>
__global__ void __launch_bounds__(kTokenThreads) combine_kernel(const Bits<D>* __restrict__ rows,
                                                                const int* __restrict__ slots,
                                                                const Bits<WD>* __restrict__ weights, long long tokens,
                                                                int top, long long h, Bits<D>* __restrict__ y,
                                                                long long y_stride) {
    const long long c = (static_cast<long long>(blockIdx.y) * blockDim.x + threadIdx.x) * E;
    if (c >= h) return;
    for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
        float acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.0f;
        for (int j0 = 0; j0 < top; j0 += U) {
            Raw<D, E> r[U];
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int slot = j0 + u < top ? __ldg(slots + t * top + j0 + u) : -1;
                const bool kept = in_rows(slot, tokens * top);
                r[u] = kept ? load_raw_cs<D, E>(rows + static_cast<long long>(slot) * h + c) : zero_raw<D, E>();
                w[u] = !kept ? 0.0f : weights == nullptr ? 1.0f : Ty<WD>::load(__ldg(weights + t * top + j0 + u));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[E];
                unpack<D, E>(r[u], f);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(w[u], f[e], acc[e]);
            }
        }
        store_f_cs<D, E>(y + t * y_stride + c, acc);
    }
}

// A warp per assignment: a dot product needs no barrier, and a warp reads its row of `rows` in kFlight
// accesses at a time; the token's row, which the block's other warps read too, comes from L1. (A
// block per token with 4 or 8 rows in flight and block-wide sums took 199 and 241 us for 8192 tokens of
// 8 x 4096 bf16; this takes 177 us.) A lane adds every kFlight-th of its products in the same register, the
// registers and the lanes are added by trees.
constexpr int kFlight = 4;

template <int D, int WD, int E>
__global__ void __launch_bounds__(kTokenThreads) combine_backward_kernel(
    const Bits<D>* __restrict__ dy, long long dy_stride, const Bits<D>* __restrict__ rows, const int* __restrict__ slots,
    const int* __restrict__ kept, const Bits<WD>* __restrict__ weights, long long tokens, int top, long long h,
    Bits<D>* __restrict__ drows, Bits<WD>* __restrict__ dweights) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const long long n = tokens * top, first = static_cast<long long>(blockIdx.x) * warps + (threadIdx.x >> 5);
    const long long step = static_cast<long long>(gridDim.x) * warps;
    for (long long a = first; a < n; a += step) {
        const int slot = __ldg(slots + a);
        if (!in_rows(slot, n)) {
            if (dweights != nullptr && lane == 0) dweights[a] = Ty<WD>::store(0.0f);
            continue;
        }
        const float w = weights == nullptr ? 1.0f : Ty<WD>::load(__ldg(weights + a));
        const Bits<D>* g = dy + a / top * dy_stride;
        const long long at = static_cast<long long>(slot) * h;
        float dot[kFlight] = {};
        for (long long c0 = lane * E; c0 < h; c0 += 32 * kFlight * E) {
            Raw<D, E> r[kFlight], t[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                const long long c = c0 + u * 32 * E;
                r[u] = c < h && dweights != nullptr ? load_raw_cs<D, E>(rows + at + c) : zero_raw<D, E>();
                t[u] = c < h ? load_raw<D, E>(g + c) : zero_raw<D, E>();
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                const long long c = c0 + u * 32 * E;
                float f[E], d[E];
                unpack<D, E>(r[u], f);
                unpack<D, E>(t[u], d);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    dot[u] = fmaf(d[e], f[e], dot[u]);
                    d[e] *= w;
                }
                if (c < h && drows != nullptr) store_f_cs<D, E>(drows + at + c, d);
            }
        }
        if (dweights == nullptr) continue;
        const float s = warp_sum((dot[0] + dot[1]) + (dot[2] + dot[3]));
        if (lane == 0) dweights[a] = Ty<WD>::store(s);
    }
    if (drows == nullptr) return;
    for (long long i = __ldg(kept) + first; i < n; i += step)
        for (long long c = lane * E; c < h; c += 32 * E) store_raw_cs<D, E>(drows + i * h + c, zero_raw<D, E>());
}

constexpr long long kMaxBlocks = 1 << 20;

dim3 token_grid(long long tokens, long long h, int e, int threads) {
    return dim3(static_cast<unsigned>(std::min(tokens, kMaxBlocks)),
                static_cast<unsigned>(ceil_div(h, static_cast<long long>(threads) * e)));
}
int token_threads(long long h, int e, int most) {
    return static_cast<int>(std::min<long long>(most, round32(ceil_div(h, e))));
}

}  // namespace
}  // namespace ops

size_t ExpertSortWorkspace(long long n) { return sizeof(unsigned int) * ops::sort_totals(n); }

cudaError_t LaunchExpertSort(const void* ids, int ids64, long long n, int experts, int* slots, int* sources,
                             int* offsets, void* workspace, cudaStream_t stream) {
    using namespace ops;
    if (n == 0) return cudaMemsetAsync(offsets, 0, sizeof(int) * (experts + 1), stream);
    int bits = 1;
    while ((1 << bits) < experts + 1) ++bits;
    const KeySource key{ids, ids64, 0, experts, 0, 0};
    return with_bits(bits, [&](auto B) {
        constexpr int kB = decltype(B)::value;
        unsigned int* totals = static_cast<unsigned int*>(workspace);
        if (n <= kClusterSort)
            return launch_sort(expert_sort_kernel<kB, kCluster>, true, n, kB, stream, key, n, totals, slots, sources, offsets);
        const cudaError_t e =
            launch_sort(expert_sort_kernel<kB, kCount>, false, n, kB, stream, key, n, totals, slots, sources, offsets);
        if (e != cudaSuccess) return e;
        return launch_sort(expert_sort_kernel<kB, kPlace>, false, n, kB, stream, key, n, totals, slots, sources, offsets);
    });
}

cudaError_t LaunchExpertDispatch(const void* x, long long x_stride, const int* slots, const int* offsets,
                                 long long tokens, int top, int experts, long long h, void* rows, int dtype,
                                 cudaStream_t stream) {
    using namespace ops;
    if (tokens == 0 || top == 0) return cudaSuccess;
    const int size = size_of(dtype);
    const bool wide = rows16(x, x_stride, h, size) && on16(rows);
    return with_type(dtype, [&](auto D) {
        constexpr int kD = decltype(D)::value, kE = Vec<kD>::E;
        auto go = [&](auto EE) {
            constexpr int E = decltype(EE)::value;
            const int threads = token_threads(h, E, kTokenThreads);
            dispatch_kernel<kD, E><<<token_grid(tokens, h, E, threads), threads, 0, stream>>>(
                static_cast<const Bits<kD>*>(x), x_stride, slots, offsets + experts, tokens, top, h,
                static_cast<Bits<kD>*>(rows));
            return cudaGetLastError();
        };
        return wide ? go(Int<kE>{}) : go(Int<1>{});
    });
}

cudaError_t LaunchExpertCombine(const void* rows, const int* slots, const void* weights, int wdtype, long long tokens,
                                int top, long long h, void* y, long long y_stride, int dtype, cudaStream_t stream) {
    using namespace ops;
    if (tokens == 0) return cudaSuccess;
    const int size = size_of(dtype);
    const bool wide = rows16(y, y_stride, h, size) && on16(rows);
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value, kE = Vec<kD>::E;
        auto go = [&](auto EE, auto UU) {
            constexpr int E = decltype(EE)::value, U = decltype(UU)::value;
            const int threads = token_threads(h, E, kTokenThreads);
            combine_kernel<kD, kW, E, U><<<token_grid(tokens, h, E, threads), threads, 0, stream>>>(
                static_cast<const Bits<kD>*>(rows), slots, static_cast<const Bits<kW>*>(weights), tokens, top, h,
                static_cast<Bits<kD>*>(y), y_stride);
            return cudaGetLastError();
        };
        if (top <= 2) return wide ? go(Int<kE>{}, Int<2>{}) : go(Int<1>{}, Int<2>{});
        return wide ? go(Int<kE>{}, Int<8>{}) : go(Int<1>{}, Int<8>{});
    });
}

cudaError_t LaunchExpertCombineBackward(const void* dy, long long dy_stride, const void* rows, const int* slots,
                                        const int* offsets, const void* weights, int wdtype, long long tokens, int top,
                                        int experts, long long h, void* drows, void* dweights, int dtype,
                                        cudaStream_t stream) {
    using namespace ops;
    if (tokens == 0 || top == 0) return cudaSuccess;
    const int size = size_of(dtype);
    const bool wide = rows16(dy, dy_stride, h, size) && on16(rows) && (drows == nullptr || on16(drows));
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value, kE = Vec<kD>::E;
        auto go = [&](auto EE) {
            constexpr int E = decltype(EE)::value;
            const long long blocks = ceil_div(tokens * top, kTokenThreads / 32);
            combine_backward_kernel<kD, kW, E>
                <<<static_cast<unsigned>(std::min(blocks, kMaxBlocks)), kTokenThreads, 0, stream>>>(
                    static_cast<const Bits<kD>*>(dy), dy_stride, static_cast<const Bits<kD>*>(rows), slots,
                    offsets + experts, static_cast<const Bits<kW>*>(weights), tokens, top, h,
                    static_cast<Bits<kD>*>(drows), static_cast<Bits<kW>*>(dweights));
            return cudaGetLastError();
        };
        return wide ? go(Int<kE>{}) : go(Int<1>{});
    });
}

}  // namespace bccl
