// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale * table[ids[i] - first],  dtable[v] = scale * sum of dy[i] over ids[i] == first + v
//
// Gradient, three launches. (1) The positions are sorted by token (key_sort.cuh; more launches for
// more than 32768). (2) The sorted positions are cut into windows of equal length, so a token
// that is everywhere is summed by many blocks: a block adds the rows of its window in order and
// writes every token that lies wholly in it; the part of a token that runs over the window's
// edge goes to a 32-bit partial row. The same launch writes zeros to the rows that do not occur.
// (3) The partial rows of a token are added in order. Every row of dtable is written once, by
// one block, and every sum has a fixed order.
// Bound by memory: dy in, dtable out.
#include "kernels/key_sort.cuh"
#include "kernels/ops.h"

#include <algorithm>

namespace bccl {
namespace ops {
namespace {

constexpr int kThreads = 256;

// A thread copies its columns of TOKENS rows, all in flight at once: a row cannot be asked for before
// its id is there, so one row at a time leaves the memory idle (32768 rows of 8 KiB: 97 us, with four 63).
// blockDim (x, y): columns, groups of TOKENS rows.
template <int D, typename Form, int TOKENS>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const KeySource key, long long n, const Bits<D>* __restrict__ table,
                                                          long long table_stride, int h, float scale,
                                                          Bits<D>* __restrict__ out, long long out_stride) {
    constexpr int E = Vec<D>::E;
    constexpr bool ODD = Form::odd;
    const int j = blockIdx.y * blockDim.x + threadIdx.x;
    if (!ODD && j * E >= h) return;
    const long long step = static_cast<long long>(gridDim.x) * rows_per_block<Form>() * TOKENS;
    for (long long i0 = (static_cast<long long>(blockIdx.x) * rows_per_block<Form>() + row_in_block<Form>()) * TOKENS; i0 < n;
         i0 += step) {
        unsigned int row[TOKENS];
#pragma unroll
        for (int t = 0; t < TOKENS; ++t)
            row[t] = i0 + t < n ? key(i0 + t) : static_cast<unsigned int>(key.bins);
        Started<ODD> r[TOKENS];
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
            const Bits<D>* from = table + row[t] * table_stride;
            if constexpr (!ODD) {  // rows of frequent tokens stay in L1 and L2
                r[t].lo = row[t] < key.bins ? __ldg(reinterpret_cast<const uint4*>(from + j * E)) : make_uint4(0, 0, 0, 0);
            } else {
                const int c = j * E - shift_of<ODD, D>(out + (i0 + t) * out_stride);
                r[t] = start_row<ODD, D>(from, c, h, row[t] < key.bins && c < h);
            }
        }
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
            Bits<D>* to = out + (i0 + t) * out_stride;
            const int c = j * E - shift_of<ODD, D>(to);
            if (i0 + t >= n) break;
            if (ODD && c >= h) continue;
            const Raw<D, E> v = finish_row<ODD, D>(r[t], table + row[t] * table_stride, c, h, row[t] < key.bins);
            if (scale == 1.0f) {
                put_raw<ODD, D>(to, c, h, v);
            } else {
                float f[E];
                unpack<D, E>(v, f);
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = row[t] < key.bins ? f[e] * scale : 0.0f;
                put_row<ODD, D, E>(to, c, h, f);
            }
        }
    }
}

// Writes {row, position} of the n positions to b, by row; a is the other buffer between passes. A
// cluster does all passes; kCount and kPlace launches do pass `first` only.
template <int BITS, SortMode MODE>
__global__ void __launch_bounds__(1024) position_sort_kernel(const KeySource key, long long n, int first, int passes,
                                                             unsigned int* grid_totals, uint2* a, uint2* b) {
    extern __shared__ unsigned int counters[];
    const int end = MODE == kCluster ? passes : first + 1;
    for (int p = first; p < end; ++p) {
        // Buffers alternate so that the last pass writes b.
        uint2* to = ((passes - 1 - p) & 1) ? a : b;
        const uint2* from = to == a ? b : a;
        sort_pass<BITS, MODE>(
            counters, grid_totals, n, p * BITS, p == passes - 1,
            [&](long long i) {
                return p == 0 ? make_uint2(key(i), static_cast<unsigned int>(i)) : __ldcg(from + i);
            },
            [&](unsigned int place, unsigned int k, unsigned int pos) { to[place] = make_uint2(k, pos); },
            [](unsigned int, unsigned int) {});
    }
}

// Columns [c, c + E) of a row of the table's gradient.
template <int OD, int E, bool ODD>
__device__ __forceinline__ void write_row(Bits<OD>* row, int c, int h, const float (&sum)[E], float scale, bool accumulate) {
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = sum[e] * scale;
    if (accumulate) {
        // Plain loads: this kernel writes the array they read.
        if (!ODD || (c >= 0 && c + E <= h)) {
            constexpr int W = Vec<OD>::E;
#pragma unroll
            for (int i = 0; i < E / W; ++i) {
                float t[W];
                Vec<OD>::unpack(*(reinterpret_cast<const uint4*>(row + c) + i), t);
#pragma unroll
                for (int e = 0; e < W; ++e) f[i * W + e] = fmaf(sum[i * W + e], scale, t[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (c + e >= 0 && c + e < h) f[e] = fmaf(sum[e], scale, Ty<OD>::load(row[c + e]));
        }
    }
    put_row<ODD, OD, E>(row, c, h, f);
}

constexpr int kMaxWindow = 128;
constexpr int kFlight = 8;  // rows of dy in flight per thread

struct WindowArgs {
    const uint2* sorted;
    long long n, rows;
    int h;
    int window;
    long long windows;
    float* partial;      // [windows][2][width]: a token that came from the left; one that goes on to the right
    long long width;     // by accesses: columns of a row begin at its shift
    float scale;
    int accumulate;
    int tile;            // rows that a block clears at a time
    int window_blocks;   // blocks of windows, the others clear
    int join_windows;    // windows that a block of the join looks at
    int join_columns;    // stretches of kJoinColumns accesses in a row
};

constexpr int kMaxTile = 4096;

// First of the n sorted positions whose row is at least `row`.
__device__ __forceinline__ long long first_of(const uint2* sorted, long long n, long long row) {
    long long lo = 0, hi = n;
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (__ldg(&sorted[mid].x) < row) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// Zeros for the rows of the table that do not occur among the sorted positions. The positions of a
// tile's rows set bits in shared memory. (Marking rows while sorting took longer than the sort: thousands
// of stores to the byte of a frequent token.)
template <int OD, int E, bool ODD>
__device__ __forceinline__ void clear_absent(const WindowArgs& a, int j, Bits<OD>* dtable) {
    __shared__ unsigned int present[kMaxTile / 32];
    __shared__ long long range[2];
    const int id = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
    float zero[E];
#pragma unroll
    for (int e = 0; e < E; ++e) zero[e] = 0.0f;
    const long long tiles = (a.rows + a.tile - 1) / a.tile;
    for (long long t = static_cast<long long>(blockIdx.x) - a.window_blocks; t < tiles; t += gridDim.x - a.window_blocks) {
        const long long r0 = t * a.tile;
        const int count = static_cast<int>(min(static_cast<long long>(a.tile), a.rows - r0));
        for (int i = id; i < (count + 31) / 32; i += threads) present[i] = 0;
        for (int i = id; i < 2; i += threads) range[i] = first_of(a.sorted, a.n, i == 0 ? r0 : r0 + count);
        __syncthreads();
        for (long long i = range[0] + id; i < range[1]; i += threads) {
            const unsigned int row = __ldg(&a.sorted[i].x);
            // A token's first position is enough.
            if (i == range[0] || __ldg(&a.sorted[i - 1].x) != row)
                atomicOr(&present[(row - r0) >> 5], 1u << ((row - r0) & 31));
        }
        __syncthreads();
        for (int r = threadIdx.y; r < count; r += blockDim.y) {
            if (present[r >> 5] >> (r & 31) & 1) continue;
            Bits<OD>* row = dtable + (r0 + r) * a.h;
            const int c = j * E - shift_of<ODD, OD>(row);
            if (c < a.h) put_row<ODD, OD, E>(row, c, a.h, zero);
        }
        __syncthreads();
    }
}

// blockDim (x, y): columns, windows. blockIdx.x < window_blocks: windows of sorted positions; beyond:
// rows to clear. blockIdx.y: columns.
template <int D, int OD, typename Form>
__global__ void __launch_bounds__(kThreads) window_kernel(const WindowArgs a, const Bits<D>* __restrict__ dy,
                                                          long long dy_stride, Bits<OD>* __restrict__ dtable) {
    constexpr int E = Vec<D>::E;
    constexpr bool ODD = Form::odd;
    extern __shared__ uint2 items[];  // [blockDim.y][window + 2]: the windows and their neighbours on either side
    const int j = blockIdx.y * blockDim.x + threadIdx.x, h = a.h;
    if (static_cast<int>(blockIdx.x) >= a.window_blocks) {
        clear_absent<OD, E, ODD>(a, j, dtable);
        return;
    }
    const long long w = static_cast<long long>(blockIdx.x) * rows_per_block<Form>() + row_in_block<Form>();
    const long long w0 = w * a.window;
    const int count = static_cast<int>(max(0ll, min(a.n - w0, static_cast<long long>(a.window))));
    uint2* it = items + row_in_block<Form>() * (a.window + 2) + 1;
    for (int i = threadIdx.x; i < count + 2; i += blockDim.x) {
        const long long k = w0 + i - 1;
        it[i - 1] = k >= 0 && k < a.n ? __ldg(a.sorted + k) : make_uint2(0xffffffffu, 0);
    }
    __syncthreads();
    if (!ODD && j * E >= h) return;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    bool from_left = count > 0 && it[-1].x == it[0].x;
    constexpr int U = ODD ? kFlight / 2 : kFlight;  // putting ODD rows together takes registers
    for (int i0 = 0; i0 < count; i0 += U) {
        Started<ODD> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint2 item = i0 + u < count ? it[i0 + u] : make_uint2(0xffffffffu, 0);
            const bool in = item.x < a.rows;
            const int c = j * E - (in ? shift_of<ODD, OD>(dtable + static_cast<long long>(item.x) * h) : 0);
            r[u] = start_row<ODD, D>(dy + static_cast<long long>(item.y) * dy_stride, c, h, in && (!ODD || c < h));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u;
            if (i >= count) break;
            const unsigned int row = it[i].x;
            if (row >= a.rows) return;  // sorted last: nothing but dropped positions follows
            Bits<OD>* to = dtable + static_cast<long long>(row) * h;
            const int c = j * E - shift_of<ODD, OD>(to);
            float f[E];
            unpack<D, E>(finish_row<ODD, D>(r[u], dy + static_cast<long long>(it[i].y) * dy_stride, c, h, c < h), f);
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += f[e];
            if (it[i + 1].x == row && i + 1 < count) continue;
            const bool to_right = it[i + 1].x == row;
            if (ODD && c >= h) {
                // nothing of this row in this thread
            } else if (from_left || to_right) {
                float* p = a.partial + (w * 2 + (from_left ? 0 : 1)) * a.width + j * E;
                store_f<kF32, E>(reinterpret_cast<Bits<kF32>*>(p), sum);
            } else {
                write_row<OD, E, ODD>(to, c, h, sum, a.scale, a.accumulate != 0);
            }
            from_left = false;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] = 0.0f;
        }
    }
}

// The window in which a token begins that runs over its right edge adds the token's partial rows. A
// block looks at up to kJoinWindows windows at once (fewer where that leaves SMs idle), most of which have
// nothing to join, for kJoinColumns accesses of columns; its kJoinParts rows of threads add consecutive shares of the partial rows and
// are then added in order. (With one row of threads a token in 737 windows took 52 us, so 24.)
constexpr int kJoinColumns = 32, kJoinParts = 8, kJoinWindows = 8, kJoinFlight = 4;

template <int OD, int E, bool ODD>
__global__ void __launch_bounds__(kJoinColumns * kJoinParts) join_kernel(const WindowArgs a, Bits<OD>* __restrict__ dtable) {
    __shared__ float parts[kJoinParts][kJoinColumns][E + 1];
    __shared__ long long last_of[kJoinWindows];  // last window of the token that begins in each and goes on, or -1
    const long long w0 = static_cast<long long>(blockIdx.x) * a.join_windows;
    if (threadIdx.y == 0 && threadIdx.x < a.join_windows) {
        const long long w = w0 + threadIdx.x, begin = w * a.window, end = begin + a.window;
        long long last = -1;
        if (end < a.n) {  // windows but the last are full
            const unsigned int row = __ldg(&a.sorted[end - 1].x), right = __ldg(&a.sorted[end].x);
            const unsigned int left = begin > 0 ? __ldg(&a.sorted[begin - 1].x) : 0xffffffffu;
            if (row < a.rows && right == row && left != row) {  // left == row: it began in an earlier window
                // The last window whose first position has the token: mostly the next one, so search
                // in growing steps.
                long long step = 1;
                last = w + 1;
                while (last + step < a.windows && __ldg(&a.sorted[(last + step) * a.window].x) == row) {
                    last += step;
                    step *= 2;
                }
                for (; step > 1; step /= 2) {
                    const long long mid = last + step / 2;
                    if (mid < a.windows && __ldg(&a.sorted[mid * a.window].x) == row) last = mid;
                }
            }
        }
        last_of[threadIdx.x] = last;
    }
    __syncthreads();
    for (int i = 0; i < a.join_windows; ++i) {
        const long long w = w0 + i, last = last_of[i];
        if (last < 0) continue;
        // Rows near 2^23 elements have more stretches of columns than a grid has blocks in y.
        for (int stretch = blockIdx.y; stretch < a.join_columns; stretch += gridDim.y) {
            const int j = stretch * kJoinColumns + threadIdx.x;
            float sum[E];
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] = 0.0f;
            const long long share = (last - w + kJoinParts) / kJoinParts;  // of last - w + 1 partial rows
            const long long k1 = min(last + 1, w + (threadIdx.y + 1) * share);
            if (j * E < a.width) {
                for (long long k0 = w + threadIdx.y * share; k0 < k1; k0 += kJoinFlight) {
                    float f[kJoinFlight][E];
#pragma unroll
                    for (int u = 0; u < kJoinFlight; ++u)
                        if (k0 + u < k1)
                            load_f<kF32, E>(reinterpret_cast<const Bits<kF32>*>(
                                                a.partial + ((k0 + u) * 2 + (k0 + u == w ? 1 : 0)) * a.width + j * E),
                                            f[u]);
#pragma unroll
                    for (int u = 0; u < kJoinFlight; ++u) {
                        if (k0 + u >= k1) break;
#pragma unroll
                        for (int e = 0; e < E; ++e) sum[e] += f[u][e];
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) parts[threadIdx.y][threadIdx.x][e] = sum[e];
            __syncthreads();
            const unsigned int row = __ldg(&a.sorted[(w + 1) * a.window].x);
            Bits<OD>* to = dtable + static_cast<long long>(row) * a.h;
            const int c = j * E - shift_of<ODD, OD>(to);
            if (threadIdx.y == 0 && c < a.h) {
                for (int p = 1; p < kJoinParts; ++p) {
#pragma unroll
                    for (int e = 0; e < E; ++e) sum[e] += parts[p][threadIdx.x][e];
                }
                write_row<OD, E, ODD>(to, c, a.h, sum, a.scale, a.accumulate != 0);
            }
            __syncthreads();
        }
    }
}

// Positions per window: long ones make fewer partial rows, short ones more threads (150000 fill the
// GPU's SMs by half).
int window_of(long long n, long long h) {
    int w = 8;
    while (w < kMaxWindow && n / (2 * w) * ceil_div(h, 8) >= 150000) w *= 2;
    return w;
}

size_t align16(size_t v) { return (v + 15) / 16 * 16; }
long long partial_width(long long h) { return (h + 14) / 8 * 8; }  // accesses of 4 or 8 columns at any shift

}  // namespace
}  // namespace ops

cudaError_t LaunchEmbeddingForward(const EmbeddingArgs& a, const void* table, long long table_stride, float scale,
                                   void* out, long long out_stride, int dtype, cudaStream_t stream) {
    using namespace ops;
    if (a.n == 0 || a.h == 0) return cudaSuccess;
    const int size = size_of(dtype);
    const bool odd = !rows16(table, table_stride, a.h, size) || !rows16(out, out_stride, a.h, size);
    const KeySource key{a.ids, a.ids64, a.first, a.rows, 0, 0};
    return with_type(dtype, [&](auto D) {
        constexpr int kD = decltype(D)::value;
        return with_form(odd, a.h, Vec<kD>::E, kThreads, [&](auto form, long long wide, BlockShape b) {
            auto go = [&](auto TT) {
                constexpr int T = decltype(TT)::value;
                const dim3 grid(static_cast<unsigned>(std::min<long long>(ceil_div(a.n, T * b.y), 1 << 20)),
                                static_cast<unsigned>(ceil_div(wide, b.x)));
                lookup_kernel<kD, decltype(form), T><<<grid, dim3(b.x, b.y), 0, stream>>>(
                    key, a.n, static_cast<const Bits<kD>*>(table), table_stride, static_cast<int>(a.h), scale,
                    static_cast<Bits<kD>*>(out), out_stride);
                return cudaGetLastError();
            };
            // Few accesses: one row each, on as many SMs as there are.
            return a.n * wide < 16ll * kThreads * sm_count() ? go(Int<1>{}) : go(Int<decltype(form)::odd ? 2 : 4>{});
        });
    });
}

size_t EmbeddingBackwardWorkspace(long long n, long long h) {
    using namespace ops;
    const long long windows = ceil_div(n, window_of(n, h));
    return 2 * align16(sizeof(uint2) * static_cast<size_t>(n)) + align16(sizeof(unsigned int) * sort_totals(n)) +
           align16(sizeof(float) * 2 * static_cast<size_t>(windows) * static_cast<size_t>(partial_width(h)));
}

cudaError_t LaunchEmbeddingBackward(const EmbeddingArgs& a, const void* dy, long long dy_stride, void* dtable,
                                    float scale, long long skip, bool has_skip, bool accumulate, int dtype,
                                    int out_dtype, void* workspace, cudaStream_t stream) {
    using namespace ops;
    if (a.rows == 0 || a.h == 0) return cudaSuccess;
    if (a.n == 0) {
        if (accumulate) return cudaSuccess;
        return cudaMemsetAsync(dtable, 0, static_cast<size_t>(a.rows) * a.h * size_of(out_dtype), stream);
    }
    char* ws = static_cast<char*>(workspace);
    uint2* buf_a = reinterpret_cast<uint2*>(ws);
    ws += align16(sizeof(uint2) * static_cast<size_t>(a.n));
    uint2* buf_b = reinterpret_cast<uint2*>(ws);
    ws += align16(sizeof(uint2) * static_cast<size_t>(a.n));
    unsigned int* totals = reinterpret_cast<unsigned int*>(ws);
    ws += align16(sizeof(unsigned int) * sort_totals(a.n));
    float* partial = reinterpret_cast<float*>(ws);

    int key_bits = 1;
    while (key_bits < 31 && (1ll << key_bits) < a.rows + 1) ++key_bits;
    const int passes = static_cast<int>(ceil_div(key_bits, kSortMaxBits));
    const int bits = static_cast<int>(ceil_div(key_bits, passes));
    const KeySource key{a.ids, a.ids64, a.first, a.rows, skip, has_skip ? 1 : 0};
    const cudaError_t e = with_bits(bits, [&](auto B) {
        constexpr int kB = decltype(B)::value;
        if (a.n <= kClusterSort)
            return launch_sort(position_sort_kernel<kB, kCluster>, true, a.n, kB, stream, key, a.n, 0, passes, totals, buf_a,
                               buf_b);
        for (int p = 0; p < passes; ++p) {
            cudaError_t err = launch_sort(position_sort_kernel<kB, kCount>, false, a.n, kB, stream, key, a.n, p, passes, totals,
                                          buf_a, buf_b);
            if (err == cudaSuccess)
                err = launch_sort(position_sort_kernel<kB, kPlace>, false, a.n, kB, stream, key, a.n, p, passes, totals, buf_a,
                                  buf_b);
            if (err != cudaSuccess) return err;
        }
        return cudaSuccess;
    });
    if (e != cudaSuccess) return e;

    WindowArgs args{};
    args.sorted = buf_b;
    args.n = a.n;
    args.rows = a.rows;
    args.h = static_cast<int>(a.h);
    args.window = window_of(a.n, a.h);
    args.windows = ceil_div(a.n, args.window);
    args.partial = partial;
    args.width = partial_width(a.h);
    args.scale = scale;
    args.accumulate = accumulate ? 1 : 0;
    const bool odd = !rows16(dy, dy_stride, a.h, size_of(dtype)) || !rows16(dtable, a.h, a.h, size_of(out_dtype));
    return with_types(dtype, out_dtype, [&](auto D, auto O) {
        constexpr int kD = decltype(D)::value, kO = decltype(O)::value, E = Vec<kD>::E;
        return with_form(odd, a.h, E, kThreads, [&](auto form, long long wide, BlockShape b) {
            using Form = decltype(form);
            b.y = std::min<int>(b.y, 40 * 1024 / (sizeof(uint2) * (args.window + 2)));  // windows in shared memory
            const unsigned cols = static_cast<unsigned>(ceil_div(wide, b.x));
            // Tiles of about 128 KiB, a block each, so that blocks whose rows mostly occur make room
            // for others (8 persistent blocks per SM with equal shares: 228 us for 32768 tokens, 128256
            // rows of 8 KiB; tiles 196 us), but two blocks per SM at least.
            WindowArgs w = args;
            const long long bytes = std::min<long long>(a.h, static_cast<long long>(b.x) * E) * sizeof(Bits<kO>);
            const long long tile = std::min(std::max(32ll, 128 * 1024 / bytes),
                                            ceil_div(a.rows, std::max(1ll, static_cast<long long>(sm_count()) * 2 / cols)));
            w.tile = static_cast<int>(std::min<long long>(kMaxTile, std::max(1ll, tile)));
            const long long clear = accumulate ? 0 : std::min(1ll << 20, ceil_div(a.rows, w.tile));
            w.window_blocks = static_cast<int>(ceil_div(w.windows, b.y));
            w.join_columns = static_cast<int>(ceil_div(wide, kJoinColumns));
            w.join_windows = static_cast<int>(
                std::min<long long>(kJoinWindows, std::max(1ll, w.windows * w.join_columns / (8 * sm_count()))));
            const size_t smem = sizeof(uint2) * b.y * (w.window + 2);
            window_kernel<kD, kO, Form>
                <<<dim3(static_cast<unsigned>(w.window_blocks + clear), cols), dim3(b.x, b.y), smem, stream>>>(
                    w, static_cast<const Bits<kD>*>(dy), dy_stride, static_cast<Bits<kO>*>(dtable));
            cudaError_t err = cudaGetLastError();
            if (err != cudaSuccess || w.windows == 1) return err;
            const dim3 grid(static_cast<unsigned>(ceil_div(w.windows - 1, w.join_windows)),
                            static_cast<unsigned>(std::min(w.join_columns, 65535)));
            join_kernel<kO, E, Form::odd><<<grid, dim3(kJoinColumns, kJoinParts), 0, stream>>>(w, static_cast<Bits<kO>*>(dtable));
            return cudaGetLastError();
        });
    });
}

}  // namespace bccl
