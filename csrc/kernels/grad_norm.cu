// Global gradient norm over many tensors, and clipping by it.
//
//   norm = sqrt(sum_t sum_i g_ti^2),  c = min(1, max_norm / (norm + eps)),  out = c * g
//
// Three launches for up to kMaxTensors tensors: the squares (a block per 32 KiB chunk writes one
// partial sum), their sum (one block), the scaling (a block per chunk again). No atomics, every sum
// in a fixed order, no state between launches.
// Bound by memory: bytes in for the norm, bytes in and out again where c < 1. A block per chunk
// and not a persistent grid: reading 1.74 GB took 238 us against 243 to 253 us for 592 to 2368
// persistent blocks, reading and writing it 508 us against 546 to 589 us.
#include "kernels/ops.h"
#include "kernels/ops_common.cuh"

#include <algorithm>
#include <mutex>

namespace bccl {
namespace ops {

int sm_count() {
    static std::mutex mu;
    static int sms[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    std::lock_guard<std::mutex> lk(mu);
    if (sms[dev] == 0 && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        sms[dev] = 148;
    return sms[dev];
}

namespace {

constexpr int kMaxTensors = 1024;  // per launch: 28 bytes each, within the 32 KiB of launch parameters
constexpr int kThreads = 256;
constexpr int kUnroll = 8;         // 16-byte loads in flight per thread
constexpr int kChunkVecs = kThreads * kUnroll;  // a chunk is 32 KiB of input

// Tensors are cut into chunks that start on 16-byte boundaries of the input (the first chunk
// holds the elements before the first boundary too). start[i] is the first chunk of tensor i.
template <int N> struct Table {
    const void* in[N];
    void* out[N];
    unsigned long long count[N];
    unsigned int start[N + 1];
    int n;
};

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, unsigned int chunk) {
    int lo = 0, hi = t.n;  // start[lo] <= chunk < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.start[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

// Calls vec(p) for whole 16-byte groups of the chunk and one(i) for single elements at the
// tensor's ends; `base` is the tensor's address rounded down to 16 bytes, in elements `skew`
// before its first.
template <int D> struct ChunkView {
    const Bits<D>* base;
    long long first, last;  // elements of the tensor, relative to base: [first, last)
    long long lo, hi;       // 16-byte groups of this chunk that hold any of them
    static constexpr int E = Vec<D>::E;
    __device__ ChunkView(const void* p, unsigned long long n, unsigned int chunk) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        base = reinterpret_cast<const Bits<D>*>(a & ~static_cast<uintptr_t>(15));
        first = static_cast<long long>((a & 15) / sizeof(Bits<D>));
        last = first + static_cast<long long>(n);
        lo = static_cast<long long>(chunk) * kChunkVecs;
        const long long groups = (last + E - 1) / E;
        hi = lo + kChunkVecs < groups ? lo + kChunkVecs : groups;
    }
    __device__ bool whole(long long v) const { return v * E >= first && (v + 1) * E <= last; }
};

template <int THREADS>
__device__ __forceinline__ double block_sum_f64(double v) {
    __shared__ double buf[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < THREADS / 32 ? buf[threadIdx.x & 31] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A thread adds its at most 64 squares in 32 bits, everything beyond is added in 64: the sum's
// error does not grow with the number of elements.
template <int D, int N>
__global__ void __launch_bounds__(kThreads, 4) squares_kernel(const __grid_constant__ Table<N> t, double* partials) {
    constexpr int E = Vec<D>::E;
    const int i = tensor_of(t, blockIdx.x);
    const ChunkView<D> view(t.in[i], t.count[i], blockIdx.x - t.start[i]);
    Raw<D, E> r[kUnroll];
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long long v = view.lo + u * kThreads + threadIdx.x;
        r[u] = v < view.hi && view.whole(v) ? load_raw<D, E>(view.base + v * E) : zero_raw<D, E>();
    }
    // The first and last group of a tensor may hold other tensors' elements too.
    if (threadIdx.x < 2) {
        const long long v = threadIdx.x == 0 ? view.lo : view.hi - 1;
        if (!view.whole(v) && (threadIdx.x == 0 || v != view.lo)) {
            for (long long k = max(view.first, v * E); k < min(view.last, (v + 1) * E); ++k) {
                const float a = Ty<D>::load(__ldg(view.base + k));
                s = fmaf(a, a, s);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        float a[E];
        unpack<D, E>(r[u], a);
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(a[e], a[e], s);
    }
    const double total = block_sum_f64<kThreads>(static_cast<double>(s));
    if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

constexpr int kFoldThreads = 1024;

__global__ void __launch_bounds__(kFoldThreads) fold_kernel(const double* __restrict__ partials, unsigned int n,
                                                            int accumulate, double* sum) {
    double s = 0.0;
#pragma unroll 8
    for (unsigned int i = threadIdx.x; i < n; i += kFoldThreads) s += partials[i];
    s = block_sum_f64<kFoldThreads>(s);
    if (threadIdx.x == 0) *sum = accumulate ? *sum + s : s;
}

// The blocks take the chunks from the last to the first: what the squares read last is still in
// L2 (126 MB) and is read from there. A block takes kInPlace chunks in place and one otherwise: in place
// most launches find nothing to do, and then starting the warps is all they cost (1.5 GB: 37 us with
// a block per chunk).
constexpr int kInPlace = 4;

template <int D, int O, int N>
__global__ void __launch_bounds__(kThreads, 4) clip_kernel(const __grid_constant__ Table<N> t, int in_place,
                                                           const double* __restrict__ sum, float max_norm, float eps,
                                                           float* norm_out) {
    constexpr int E = Vec<D>::E;
    // In place, a norm below the bound by more than rounding moves nothing: most steps.
    const double free_norm = static_cast<double>(max_norm) - eps;
    if (in_place && free_norm > 0.0 && *sum < free_norm * free_norm * (1.0 - 1e-6) && (blockIdx.x != 0 || norm_out == nullptr))
        return;
    const float norm = static_cast<float>(sqrt(*sum));
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const float q = max_norm / (norm + eps);
    const float c = q > 1.0f ? 1.0f : q;  // a NaN stays
    if ((in_place && c == 1.0f) || t.n == 0) return;
    const unsigned int chunks = t.start[t.n];
    for (unsigned int k = blockIdx.x; k < chunks; k += gridDim.x) {
        const unsigned int chunk = chunks - 1 - k;
        const int i = tensor_of(t, chunk);
        const ChunkView<D> view(t.in[i], t.count[i], chunk - t.start[i]);
        Bits<O>* out = static_cast<Bits<O>*>(t.out[i]) - view.first;  // indexed like base
        const bool wide = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
        Raw<D, E> r[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long v = view.lo + u * kThreads + threadIdx.x;
            if (v < view.hi && view.whole(v)) r[u].v = __ldcs(reinterpret_cast<const uint4*>(view.base + v * E));
        }
        if (threadIdx.x < 2) {
            const long long v = threadIdx.x == 0 ? view.lo : view.hi - 1;
            if (!view.whole(v) && (threadIdx.x == 0 || v != view.lo))
                for (long long j = max(view.first, v * E); j < min(view.last, (v + 1) * E); ++j)
                    out[j] = Ty<O>::store(Ty<D>::load(view.base[j]) * c);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long v = view.lo + u * kThreads + threadIdx.x;
            if (v < view.hi && view.whole(v)) {
                float a[E];
                unpack<D, E>(r[u], a);
#pragma unroll
                for (int e = 0; e < E; ++e) a[e] *= c;
                if (wide) {
                    store_f_cs<O, E>(out + v * E, a);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) out[v * E + e] = Ty<O>::store(a[e]);
                }
            }
        }
    }
}

size_t chunks_of(const void* p, size_t count, int size) {
    const size_t skew = (reinterpret_cast<uintptr_t>(p) & 15) / size, width = static_cast<size_t>(kChunkVecs) * (16 / size);
    return (skew + count + width - 1) / width;
}

// Fills a table from tensors [i, ...) until it is full; returns the next tensor. A launch holds
// fewer than 2^31 chunks (64 TB).
template <int N>
int fill(Table<N>& t, const void* const* in, void* const* out, const size_t* counts, int i, int n, int size) {
    size_t start = 0;
    t.n = 0;
    for (; i < n && t.n < N; ++i) {
        if (counts[i] == 0) continue;
        const size_t chunks = chunks_of(in[i], counts[i], size);
        if (start + chunks > INT_MAX) return -1;
        t.in[t.n] = in[i];
        t.out[t.n] = out != nullptr ? out[i] : nullptr;
        t.count[t.n] = counts[i];
        t.start[t.n++] = static_cast<unsigned int>(start);
        start += chunks;
    }
    t.start[t.n] = static_cast<unsigned int>(start);
    return i;
}

template <int N>
cudaError_t squares(const void* const* in, const size_t* counts, int n, int dtype, bool accumulate, double* sum,
                    double* partials, cudaStream_t s) {
    Table<N> t;
    int i = 0;
    unsigned int done = 0;  // partial sums written
    do {
        i = fill(t, in, static_cast<void* const*>(nullptr), counts, i, n, size_of(dtype));
        if (i < 0) return cudaErrorInvalidValue;
        if (t.n == 0) continue;
        const cudaError_t e = with_type(dtype, [&](auto D) {
            squares_kernel<decltype(D)::value, N><<<t.start[t.n], kThreads, 0, s>>>(t, partials + done);
            return cudaGetLastError();
        });
        if (e != cudaSuccess) return e;
        done += t.start[t.n];
    } while (i < n);
    fold_kernel<<<1, kFoldThreads, 0, s>>>(partials, done, accumulate ? 1 : 0, sum);
    return cudaGetLastError();
}

template <int N>
cudaError_t clip(const void* const* in, void* const* out, const size_t* counts, int n, int dtype, int out_dtype,
                 const double* sum, float max_norm, float eps, float* norm, cudaStream_t s) {
    int in_place = 1;
    for (int i = 0; i < n; ++i) in_place &= in[i] == out[i];
    Table<N> t;
    int i = 0;
    do {
        i = fill(t, in, out, counts, i, n, size_of(dtype));
        if (i < 0) return cudaErrorInvalidValue;
        if (t.n == 0 && norm == nullptr) continue;
        const unsigned int grid = std::max(1u, in_place ? (t.start[t.n] + kInPlace - 1) / kInPlace : t.start[t.n]);
        const cudaError_t e = with_types(dtype, out_dtype, [&](auto D, auto O) {
            clip_kernel<decltype(D)::value, decltype(O)::value, N>
                <<<grid, kThreads, 0, s>>>(t, in_place, sum, max_norm, eps, norm);
            return cudaGetLastError();
        });
        if (e != cudaSuccess) return e;
        norm = nullptr;
    } while (i < n);
    return cudaSuccess;
}

// Tensors of a launch: the whole table is copied into the launch, so short lists take a short one.
template <typename F>
cudaError_t with_table(int n, F&& f) {
    if (n <= 32) return f(Int<32>{});
    if (n <= 256) return f(Int<256>{});
    return f(Int<kMaxTensors>{});
}

}  // namespace
}  // namespace ops

size_t GradSquaresWorkspace(const void* const* grads, const size_t* counts, int n, int dtype) {
    size_t chunks = 1;
    for (int i = 0; i < n; ++i)
        if (counts[i] > 0) chunks += ops::chunks_of(grads[i], counts[i], ops::size_of(dtype));
    return chunks * sizeof(double);
}

cudaError_t LaunchGradSquares(const void* const* grads, const size_t* counts, int n, int dtype, bool accumulate,
                              double* sum, void* workspace, cudaStream_t stream) {
    return ops::with_table(n, [&](auto N) {
        return ops::squares<decltype(N)::value>(grads, counts, n, dtype, accumulate, sum, static_cast<double*>(workspace),
                                                stream);
    });
}

cudaError_t LaunchGradClip(const void* const* grads, void* const* outs, const size_t* counts, int n, int dtype,
                           int out_dtype, const double* sum, float max_norm, float eps, float* norm, cudaStream_t stream) {
    return ops::with_table(n, [&](auto N) {
        return ops::clip<decltype(N)::value>(grads, outs, counts, n, dtype, out_dtype, sum, max_norm, eps, norm, stream);
    });
}

}  // namespace bccl
