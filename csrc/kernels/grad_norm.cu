// Global gradient norm over many tensors, and clipping by it.
//
//   norm = sqrt(sum_t sum_i g_ti^2),  c = min(1, max_norm / (norm + eps)),  out = c * g
//
// Two launches whatever the number of tensors (up to kMaxTensors in a launch's parameters):
// the squares, then the scaling, whose blocks each add the first launch's partial sums up again
// in a fixed order (592 doubles from L2) instead of waiting for one block to do it. No atomics,
// so the norm does not depend on timing, and no state between launches.
// Bound by memory: bytes in for the norm, bytes in and out again where c < 1.
#include "bccl/ops.h"
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

constexpr int kMaxTensors = 1024;      // per launch: 24 bytes each, within the 32 KiB of launch parameters
constexpr int kThreads = 256;
constexpr int kUnroll = 8;             // 16-byte loads in flight per thread
constexpr int kChunkVecs = kThreads * kUnroll;  // a chunk is 32 KiB of input
constexpr int kGrid = BCCL_GRAD_PARTIALS;       // 4 blocks of 256 on each of 148 SMs: 128 KiB in flight per SM

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

__device__ __forceinline__ double block_sum_f64(double v, double* buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < kThreads / 32 ? buf[threadIdx.x & 31] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A thread adds the squares of one chunk in 32 bits (at most 8 groups of 8 elements) and chunks
// in 64 bits: the sum's error does not grow with the number of elements.
template <int D, int N>
__global__ void __launch_bounds__(kThreads, 4) squares_kernel(const __grid_constant__ Table<N> t, double* partials,
                                                              int accumulate) {
    constexpr int E = Vec<D>::E;
    __shared__ double buf[32];
    const unsigned int chunks = t.start[t.n];
    double total = 0.0;
    for (unsigned int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const ChunkView<D> view(t.in[i], t.count[i], c - t.start[i]);
        Raw<D, E> r[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long v = view.lo + u * kThreads + threadIdx.x;
            r[u] = v < view.hi && view.whole(v) ? load_raw<D, E>(view.base + v * E) : zero_raw<D, E>();
        }
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float a[E];
            unpack<D, E>(r[u], a);
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(a[e], a[e], s);
        }
        // The first and last group of a tensor may hold other tensors' elements too.
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long v = view.lo + u * kThreads + threadIdx.x;
            if (v < view.hi && !view.whole(v)) {
                for (int e = 0; e < E; ++e) {
                    const long long k = v * E + e;
                    if (k >= view.first && k < view.last) {
                        const float a = Ty<D>::load(__ldg(view.base + k));
                        s = fmaf(a, a, s);
                    }
                }
            }
        }
        total += static_cast<double>(s);
    }
    total = block_sum_f64(total, buf);
    if (threadIdx.x == 0) partials[blockIdx.x] = accumulate ? partials[blockIdx.x] + total : total;
    if (!accumulate && blockIdx.x == 0)
        for (int b = gridDim.x + threadIdx.x; b < kGrid; b += kThreads) partials[b] = 0.0;
}

// The blocks walk the chunks from the last to the first: what the squares read last is still in
// L2 (126 MB) and is read from there.
template <int D, int O, int N>
__global__ void __launch_bounds__(kThreads, 4) clip_kernel(const __grid_constant__ Table<N> t,
                                                           const double* __restrict__ partials, float max_norm, float eps,
                                                           float* norm_out) {
    constexpr int E = Vec<D>::E;
    __shared__ double buf[32];
    double sum = 0.0;
    for (int b = threadIdx.x; b < kGrid; b += kThreads) sum += partials[b];
    sum = block_sum_f64(sum, buf);
    const float norm = static_cast<float>(sqrt(sum));
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const float q = max_norm / (norm + eps);
    const float c = q > 1.0f ? 1.0f : q;  // a NaN stays
    const unsigned int chunks = t.start[t.n];
    for (unsigned int k = blockIdx.x; k < chunks; k += gridDim.x) {
        const unsigned int chunk = chunks - 1 - k;
        const int i = tensor_of(t, chunk);
        if (c == 1.0f && t.in[i] == t.out[i]) continue;
        const ChunkView<D> view(t.in[i], t.count[i], chunk - t.start[i]);
        Bits<O>* out = static_cast<Bits<O>*>(t.out[i]) - view.first;  // indexed like base
        const bool wide = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
        Raw<D, E> r[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long v = view.lo + u * kThreads + threadIdx.x;
            if (v < view.hi && view.whole(v)) {
                if constexpr (E > 1) r[u].v = __ldcs(reinterpret_cast<const uint4*>(view.base + v * E));
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long v = view.lo + u * kThreads + threadIdx.x;
            if (v >= view.hi) continue;
            if (view.whole(v)) {
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
            } else {
                for (int e = 0; e < E; ++e) {
                    const long long j = v * E + e;
                    if (j >= view.first && j < view.last) out[j] = Ty<O>::store(Ty<D>::load(view.base[j]) * c);
                }
            }
        }
    }
}

// Fills a table from tensors [i, ...) until it is full; returns the next tensor.
template <int N>
int fill(Table<N>& t, const void* const* in, void* const* out, const size_t* counts, int i, int n, int size) {
    unsigned int start = 0;
    t.n = 0;
    for (; i < n && t.n < N; ++i) {
        if (counts[i] == 0) continue;
        const size_t skew = (reinterpret_cast<uintptr_t>(in[i]) & 15) / size;
        const size_t chunks = (skew + counts[i] + kChunkVecs * (16 / size) - 1) / (kChunkVecs * (16 / size));
        if (chunks > UINT_MAX - start) {
            if (t.n == 0) return -1;
            break;
        }
        t.in[t.n] = in[i];
        t.out[t.n] = out != nullptr ? out[i] : nullptr;
        t.count[t.n] = counts[i];
        t.start[t.n++] = start;
        start += static_cast<unsigned int>(chunks);
    }
    t.start[t.n] = start;
    return i;
}

template <int N>
cudaError_t squares(const void* const* in, const size_t* counts, int n, int dtype, bool accumulate, double* partials,
                    cudaStream_t s) {
    Table<N> t;
    int i = 0;
    do {
        i = fill(t, in, static_cast<void* const*>(nullptr), counts, i, n, size_of(dtype));
        if (i < 0) return cudaErrorInvalidValue;
        const int grid = static_cast<int>(std::min<unsigned int>(std::max(1u, t.start[t.n]), kGrid));
        const cudaError_t e = with_type(dtype, [&](auto D) {
            squares_kernel<decltype(D)::value, N><<<grid, kThreads, 0, s>>>(t, partials, accumulate ? 1 : 0);
            return cudaGetLastError();
        });
        if (e != cudaSuccess) return e;
        accumulate = true;
    } while (i < n);
    return cudaSuccess;
}

template <int N>
cudaError_t clip(const void* const* in, void* const* out, const size_t* counts, int n, int dtype, int out_dtype,
                 const double* partials, float max_norm, float eps, float* norm, cudaStream_t s) {
    Table<N> t;
    int i = 0;
    do {
        i = fill(t, in, out, counts, i, n, size_of(dtype));
        if (i < 0) return cudaErrorInvalidValue;
        const int grid = static_cast<int>(std::min<unsigned int>(std::max(1u, t.start[t.n]), kGrid));
        const cudaError_t e = with_types(dtype, out_dtype, [&](auto D, auto O) {
            clip_kernel<decltype(D)::value, decltype(O)::value, N><<<grid, kThreads, 0, s>>>(t, partials, max_norm, eps,
                                                                                            norm);
            return cudaGetLastError();
        });
        if (e != cudaSuccess) return e;
        norm = nullptr;
    } while (i < n);
    return cudaSuccess;
}

}  // namespace
}  // namespace ops

// Short lists travel in a short parameter block.
constexpr int kShort = 32;

cudaError_t LaunchGradSquares(const void* const* grads, const size_t* counts, int n, int dtype, bool accumulate,
                              double* partials, cudaStream_t stream) {
    if (n <= kShort) return ops::squares<kShort>(grads, counts, n, dtype, accumulate, partials, stream);
    return ops::squares<ops::kMaxTensors>(grads, counts, n, dtype, accumulate, partials, stream);
}

cudaError_t LaunchGradClip(const void* const* grads, void* const* outs, const size_t* counts, int n, int dtype,
                           int out_dtype, const double* partials, float max_norm, float eps, float* norm,
                           cudaStream_t stream) {
    if (n <= kShort)
        return ops::clip<kShort>(grads, outs, counts, n, dtype, out_dtype, partials, max_norm, eps, norm, stream);
    return ops::clip<ops::kMaxTensors>(grads, outs, counts, n, dtype, out_dtype, partials, max_norm, eps, norm, stream);
}

}  // namespace bccl
