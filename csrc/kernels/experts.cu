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

// Zeros for the rows behind the last kept one, by all blocks of a kernel: row `first`, first + step, ...
template <int D, bool ODD>
__device__ __forceinline__ void clear_tail(Bits<D>* rows, long long kept, long long n, int h, int j0, int dj, long long first,
                                           long long step) {
    constexpr int E = Vec<D>::E;
    for (long long i = max(kept, 0ll) + first; i < n; i += step) {
        Bits<D>* row = rows + i * h;
        const int shift = shift_of<ODD, D>(row);
        for (int c = j0 * E - shift; c < h; c += dj * E) put_raw<ODD, D>(row, c, h, zero_raw<D, E>());
    }
}

// blockDim (x, y): columns, tokens. blockIdx.x walks tokens, blockIdx.y columns.
template <int D, typename Form>
__global__ void __launch_bounds__(kTokenThreads) dispatch_kernel(const Bits<D>* __restrict__ x, long long x_stride,
                                                                 const int* __restrict__ slots,
                                                                 const int* __restrict__ kept, long long tokens, int top,
                                                                 int h, Bits<D>* __restrict__ rows) {
    constexpr int E = Vec<D>::E;
    constexpr bool ODD = Form::odd;
    const int j = blockIdx.y * blockDim.x + threadIdx.x;
    const long long first = static_cast<long long>(blockIdx.x) * rows_per_block<Form>() + row_in_block<Form>();
    const long long step = static_cast<long long>(gridDim.x) * rows_per_block<Form>(), n = tokens * top;
    if (!ODD && j * E >= h) return;
    for (long long t = first; t < tokens; t += step) {
        const Bits<D>* from = x + t * x_stride;
        Raw<D, E> r;
        if constexpr (!ODD) r = get_row<false, D>(from, j * E, h);
        for (int k = 0; k < top; ++k) {
            const int slot = __ldg(slots + t * top + k);
            if (!in_rows(slot, n)) continue;
            Bits<D>* to = rows + static_cast<long long>(slot) * h;
            const int c = j * E - shift_of<ODD, D>(to);
            if (ODD && c >= h) continue;
            if constexpr (ODD) r = get_row<true, D>(from, c, h);
            put_raw<ODD, D>(to, c, h, r);
        }
    }
    clear_tail<D, ODD>(rows, __ldg(kept), n, h, j, gridDim.y * blockDim.x, first, step);
}

// U rows are in flight per thread; each token's sum runs over its assignments in order.
template <int D, int WD, typename Form, int U>
__global__ void __launch_bounds__(kTokenThreads) combine_kernel(const Bits<D>* __restrict__ rows,
                                                                const int* __restrict__ slots,
                                                                const Bits<WD>* __restrict__ weights, long long tokens,
                                                                int top, int h, Bits<D>* __restrict__ y,
                                                                long long y_stride) {
    constexpr int E = Vec<D>::E;
    constexpr bool ODD = Form::odd;
    const int j = blockIdx.y * blockDim.x + threadIdx.x;
    const long long n = tokens * top;
    for (long long t = static_cast<long long>(blockIdx.x) * rows_per_block<Form>() + row_in_block<Form>(); t < tokens;
         t += static_cast<long long>(gridDim.x) * rows_per_block<Form>()) {
        Bits<D>* to = y + t * y_stride;
        const int c = j * E - shift_of<ODD, D>(to);
        if (c >= h) continue;
        float acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.0f;
        for (int k0 = 0; k0 < top; k0 += U) {
            Started<ODD> r[U];
            int slot[U];
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                slot[u] = k0 + u < top ? __ldg(slots + t * top + k0 + u) : -1;
                const bool kept = in_rows(slot[u], n);
                r[u] = start_row<ODD, D>(rows + static_cast<long long>(slot[u]) * h, c, h, kept);
                w[u] = !kept ? 0.0f : weights == nullptr ? 1.0f : Ty<WD>::load(__ldg(weights + t * top + k0 + u));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[E];
                unpack<D, E>(finish_row<ODD, D>(r[u], rows + static_cast<long long>(slot[u]) * h, c, h, in_rows(slot[u], n)), f);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(w[u], f[e], acc[e]);
            }
        }
        put_row<ODD, D, E>(to, c, h, acc);
    }
}

// A warp, or a part of one where a row is short (LANES), per assignment: a dot
// product needs no barrier, and the lanes read their row of `rows` in kFlight accesses at a time; the
// token's row, which the block's other warps read too, comes from L1. (A block per token with 4 or 8 rows
// in flight and block-wide sums took 199 and 241 us for 8192 tokens of 8 x 4096 bf16; this takes 177.) A
// lane adds every kFlight-th of its products in the same register, the registers and the lanes are added
// by trees.
constexpr int kFlight = 4;

template <int D, int WD, bool ODD, int LANES>
__global__ void __launch_bounds__(kTokenThreads) combine_backward_kernel(
    const Bits<D>* __restrict__ dy, long long dy_stride, const Bits<D>* __restrict__ rows, const int* __restrict__ slots,
    const int* __restrict__ kept, const Bits<WD>* __restrict__ weights, long long tokens, int top, int h,
    Bits<D>* __restrict__ drows, Bits<WD>* __restrict__ dweights) {
    constexpr int E = Vec<D>::E;
    constexpr int kRows = kTokenThreads / LANES;
    const int lane = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;
    const long long n = tokens * top, first = static_cast<long long>(blockIdx.x) * kRows + group;
    const long long step = static_cast<long long>(gridDim.x) * kRows;
    for (long long a0 = first - group; a0 < n; a0 += step) {  // the same trips for a whole warp
        const long long a = a0 + group;
        const int slot = a < n ? __ldg(slots + a) : -1;
        float dot[kFlight] = {};
        if (in_rows(slot, n)) {
            const float w = weights == nullptr ? 1.0f : Ty<WD>::load(__ldg(weights + a));
            const Bits<D>* g = dy + a / top * dy_stride;
            const long long at = static_cast<long long>(slot) * h;
            const int shift = drows != nullptr ? shift_of<ODD, D>(drows + at) : 0;
            for (int c0 = lane * E - shift; c0 < h; c0 += LANES * kFlight * E) {
                Raw<D, E> r[kFlight], t[kFlight];  // ODD rows put together at once: their groups take registers
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    const int c = c0 + u * LANES * E;
                    r[u] = c < h && dweights != nullptr ? get_row<ODD, D>(rows + at, c, h) : zero_raw<D, E>();
                    t[u] = c >= h ? zero_raw<D, E>() : ODD ? get_row<ODD, D>(g, c, h) : load_raw<D, E>(g + c);
                }
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    const int c = c0 + u * LANES * E;
                    float f[E], d[E];
                    unpack<D, E>(r[u], f);
                    unpack<D, E>(t[u], d);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        dot[u] = fmaf(d[e], f[e], dot[u]);
                        d[e] *= w;
                    }
                    if (c < h && drows != nullptr) put_row<ODD, D, E>(drows + at, c, h, d);
                }
            }
        }
        if (dweights == nullptr) continue;
        float s = (dot[0] + dot[1]) + (dot[2] + dot[3]);
        for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0 && a < n) dweights[a] = Ty<WD>::store(s);  // 0 for a dropped assignment
    }
    if (drows != nullptr) clear_tail<D, ODD>(drows, __ldg(kept), n, h, lane, LANES, first, step);
}

constexpr long long kMaxBlocks = 1 << 20;

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
    const bool odd = !rows16(x, x_stride, h, size) || !on16(rows);
    return with_type(dtype, [&](auto D) {
        constexpr int kD = decltype(D)::value;
        return with_form(odd, h, Vec<kD>::E, kTokenThreads, [&](auto form, long long wide, BlockShape b) {
            const dim3 grid(static_cast<unsigned>(std::min(ceil_div(tokens, b.y), kMaxBlocks)),
                            static_cast<unsigned>(ceil_div(wide, b.x)));
            dispatch_kernel<kD, decltype(form)><<<grid, dim3(b.x, b.y), 0, stream>>>(
                static_cast<const Bits<kD>*>(x), x_stride, slots, offsets + experts, tokens, top, static_cast<int>(h),
                static_cast<Bits<kD>*>(rows));
            return cudaGetLastError();
        });
    });
}

cudaError_t LaunchExpertCombine(const void* rows, const int* slots, const void* weights, int wdtype, long long tokens,
                                int top, long long h, void* y, long long y_stride, int dtype, cudaStream_t stream) {
    using namespace ops;
    if (tokens == 0) return cudaSuccess;
    const int size = size_of(dtype);
    const bool odd = !rows16(y, y_stride, h, size) || !on16(rows);
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value;
        return with_form(odd, h, Vec<kD>::E, kTokenThreads, [&](auto form, long long wide, BlockShape b) {
            const dim3 grid(static_cast<unsigned>(std::min(ceil_div(tokens, b.y), kMaxBlocks)),
                            static_cast<unsigned>(ceil_div(wide, b.x)));
            auto go = [&](auto UU) {
                combine_kernel<kD, kW, decltype(form), decltype(UU)::value><<<grid, dim3(b.x, b.y), 0, stream>>>(
                    static_cast<const Bits<kD>*>(rows), slots, static_cast<const Bits<kW>*>(weights), tokens, top,
                    static_cast<int>(h), static_cast<Bits<kD>*>(y), y_stride);
                return cudaGetLastError();
            };
            // Rows in flight; putting ODD rows together takes registers too.
            return top <= 2 ? go(Int<2>{}) : go(Int<decltype(form)::odd ? 4 : 8>{});
        });
    });
}

cudaError_t LaunchExpertCombineBackward(const void* dy, long long dy_stride, const void* rows, const int* slots,
                                        const int* offsets, const void* weights, int wdtype, long long tokens, int top,
                                        int experts, long long h, void* drows, void* dweights, int dtype,
                                        cudaStream_t stream) {
    using namespace ops;
    if (tokens == 0 || top == 0) return cudaSuccess;
    const int size = size_of(dtype);
    const bool odd = !rows16(dy, dy_stride, h, size) || !on16(rows) || (drows != nullptr && !on16(drows));
    return with_types(dtype, wdtype, [&](auto D, auto W) {
        constexpr int kD = decltype(D)::value, kW = decltype(W)::value;
        auto go = [&](auto O) {
            constexpr bool ODD = decltype(O)::value != 0;
            auto launch = [&](auto L) {
                constexpr int kLanes = decltype(L)::value;
                const long long blocks = ceil_div(tokens * top, kTokenThreads / kLanes);
                combine_backward_kernel<kD, kW, ODD, kLanes>
                    <<<static_cast<unsigned>(std::min(blocks, kMaxBlocks)), kTokenThreads, 0, stream>>>(
                        static_cast<const Bits<kD>*>(dy), dy_stride, static_cast<const Bits<kD>*>(rows), slots,
                        offsets + experts, static_cast<const Bits<kW>*>(weights), tokens, top, static_cast<int>(h),
                        static_cast<Bits<kD>*>(drows), static_cast<Bits<kW>*>(dweights));
                return cudaGetLastError();
            };
            const long long n = accesses<ODD>(h, Vec<kD>::E);
            return n <= 4 ? launch(Int<4>{}) : n <= 16 ? launch(Int<16>{}) : launch(Int<32>{});
        };
        return odd ? go(Int<1>{}) : go(Int<0>{});
    });
}

}  // namespace bccl
